"""Attention over a paged cache on the GPU against 64 bits.

Tolerance of an output: the probabilities enter the second product as bf16 (2^-8 of
each at most), a score is off by the dim + 2 cut sums of its product (each at most
2^-23 of the sum of |q k| scale), which moves a probability and the total by that
much each, exp2 and the sums of n terms add n + 8 roundings; all of that of sum p |v|.
Then one rounding to the type.  lse: the score's error and a few roundings of its own
size and of the logarithm."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def run(M, lens, queries=None, heads=8, kv_heads=2, dim=128, page=16, mxfp4=True, window=0, sinks=False, f32=False, hint=0,
        seed=0, edit=None, gap=0, first=0, behind=0, std=1.0, scale=None):
    """Compares one call; queries: of each sequence (None: one token each, no offsets)."""
    import torch

    rng = np.random.default_rng([seed, dim, heads, len(lens), mxfp4])
    table, n = K.page_tables(rng, lens, page)
    pages = K.Pages(rng, n, kv_heads, page, dim, mxfp4, std)
    offsets = None if queries is None else first + np.cumsum([0] + list(queries)).astype(np.int32)
    T = (len(lens) if queries is None else int(offsets[-1])) + behind
    q, q64 = K.values_of(rng, (T, heads, dim), False, 1.5)
    s, s64 = K.values_of(rng, (heads,), True) if sinks else (None, None)
    if edit:
        edit(pages, table)
    scale = dim ** -0.5 if scale is None else scale
    k64, v64 = pages.values()
    with np.errstate(invalid="ignore"):
        want, lse64, weight, terms = K.attention(q64, k64, v64, table, lens, offsets, scale, window, s64)
    out = torch.full(q.shape, 7.0, dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    got, lse = M.kv_attention(q, pages.device(M, gap), X.dev(table), X.dev(np.array(lens, np.int32)), scale=scale,
                              q_offsets=None if offsets is None else X.dev(offsets), max_kv_len=hint, window=window, sinks=s,
                              out=out, return_lse=True)
    got, lse = X.host(got), X.host(lse)
    mine = np.arange(T) >= 0 if offsets is None else (np.arange(T) >= first) & (np.arange(T) < offsets[-1])
    assert (got[~mine] == 7).all()
    got, lse, want, lse64, weight, terms = (a[mine] for a in (got, lse, want, lse64, weight, terms))
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad), np.argwhere(np.isnan(got) != bad)[:3]
    score = (dim + 2) * K.MFMA * terms[..., None]
    tol = weight * (X.BF16_ROUND + 2 * score + (max(lens, default=0) + 8) * K.MFMA)
    tol = tol + (X.F32_ROUND if f32 else X.BF16_ROUND) * np.abs(want) + 1e-37
    with np.errstate(invalid="ignore"):
        err = np.abs(got - want)
        over = np.where(bad | (got == want), 0, err - tol)  # (an infinity is met exactly)
    at = np.unravel_index(np.argmax(over), over.shape) if over.size else None
    assert (over <= 0).all(), (at, got[at], want[at], tol[at])
    empty = np.isneginf(lse64)
    assert np.array_equal(np.isneginf(lse), empty) and (got[empty] == 0).all()
    with np.errstate(invalid="ignore"):
        off = np.abs(lse - lse64) > score[..., 0] + 2.0 ** -21 * (1 + np.abs(lse64)) + max(lens, default=0) * K.MFMA
    assert not (off & ~empty & ~np.isnan(lse64)).any()
    return got


LENS = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129, 500]


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
def test_one_token(M, dim, mxfp4):
    run(M, LENS, dim=dim, mxfp4=mxfp4)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (7, 7), (32, 4), (16, 1), (17, 1), (40, 2), (66, 2), (130, 1)])
@pytest.mark.parametrize("mxfp4", [False, True])
def test_head_layouts(M, heads, kv_heads, mxfp4):
    run(M, [77, 0, 200], heads=heads, kv_heads=kv_heads, mxfp4=mxfp4, page=48)


@pytest.mark.parametrize("page", [16, 32, 48, 80, 512])
def test_pages(M, page):
    run(M, LENS, page=page, gap=32)
    run(M, LENS, page=page, mxfp4=False, dim=64, gap=8)


# queries of each sequence; lengths; which kernel they take is decided by rows per sequence
RAGGED = [
    ([1, 0, 3, 2], [5, 9, 3, 40]), ([5, 5, 5, 5], [5, 100, 17, 2]), ([0, 0], [3, 0]), ([8], [8]), ([8], [300]),
    ([1, 40, 0, 7], [130, 40, 5, 6]), ([70], [70]), ([33, 1, 129], [100, 64, 129]), ([200], [130]),
]


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("dim", [64, 96, 128, 192])
@pytest.mark.parametrize("queries,lens", RAGGED)
def test_many_queries(M, queries, lens, dim, mxfp4):
    run(M, lens, queries, dim=dim, mxfp4=mxfp4, first=2, behind=3)


@pytest.mark.parametrize("group", [1, 3, 5, 8, 16])
@pytest.mark.parametrize("queries", [2, 5, 13, 150])
def test_groups_of_heads(M, group, queries):
    run(M, [queries, 190, 3], [queries, queries, queries], heads=2 * group, kv_heads=2)


@pytest.mark.parametrize("window", [1, 7, 16, 33, 100])
@pytest.mark.parametrize("queries", [1, 4, 60])
def test_windows(M, window, queries):
    run(M, [queries, 40 + queries, 300], [queries] * 3, window=window, sinks=True)
    run(M, [queries, 40 + queries, 300], [queries] * 3, window=window, mxfp4=False, dim=64)


@pytest.mark.parametrize("f32", [False, True])
def test_sinks_and_types(M, f32):
    run(M, LENS, sinks=True, f32=f32)
    run(M, [0, 90, 7], [3, 90, 20], sinks=True, f32=f32, heads=16)


# the keys split over workgroups, and a hint that is too small or too large
@pytest.mark.parametrize("hint", [0, 600, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("queries", [None, [3, 1], [40, 60]])
def test_long_sequences(M, hint, queries):
    run(M, [5003, 1030], queries, heads=4, kv_heads=1, dim=64, page=64, hint=hint, sinks=hint == 600)


@pytest.mark.parametrize("dim,mxfp4", [(64, False), (128, False), (256, True), (128, True)])
def test_splits_of_every_form(M, dim, mxfp4):
    run(M, [3000, 0, 700], heads=4, kv_heads=2, dim=dim, mxfp4=mxfp4, page=32, f32=True)
    run(M, [3000, 0, 700], [9, 2, 30], heads=16, kv_heads=2, dim=dim, mxfp4=mxfp4, page=32, window=1500)
    run(M, [3000, 0, 700], [50, 2, 120], heads=4, kv_heads=1, dim=dim, mxfp4=mxfp4, page=32, f32=dim == 128)


# parts of many rows, which another kernel joins, some of them empty
@pytest.mark.parametrize("dim,mxfp4", [(32, True), (96, False), (128, True), (256, True)])
def test_joins_of_many_rows(M, dim, mxfp4):
    run(M, [900, 0, 300], [200, 20, 60], dim=dim, mxfp4=mxfp4, sinks=True, first=1, behind=2)
    run(M, [900], [300], dim=dim, mxfp4=mxfp4, window=100, f32=True)


@pytest.mark.parametrize("queries", [None, [9, 3], [100, 130]])
def test_windows_longer_than_any_sequence(M, queries):
    for window in (2 ** 31 - 1, 128, 129):
        run(M, [5, 100], queries, window=window)


@pytest.mark.parametrize("queries", [None, [2, 7], [70, 20]])
@pytest.mark.parametrize("mxfp4", [False, True])
def test_infinite_and_nan_that_are_seen(M, mxfp4, queries):
    """In keys: scores of either infinity, or NaN; in values: infinities of each dim's sign, or NaN."""
    def poison(pages, table):
        def put(x, scales, b, j, kv_head, bits):
            page, row = table[b, j // 16], j % 16
            if mxfp4:
                scales[page, kv_head, row] = 255 if bits == 0x7FC0 else 254
            else:
                x[page, kv_head, row] = bits

        put(pages.k, pages.ks, 0, 40, 0, 0x7F80)
        put(pages.v, pages.vs, 0, 95, 1, 0xFF80)
        put(pages.k, pages.ks, 1, 85, 0, 0x7FC0)
        put(pages.v, pages.vs, 1, 70, 1, 0x7FC0)

    run(M, [100, 90], queries, mxfp4=mxfp4, edit=poison)


def test_one_key_is_its_value(M):
    got = run(M, [1, 1, 1], f32=True, mxfp4=False)
    assert np.isfinite(got).all()


@pytest.mark.parametrize("queries", [None, [2, 7], [70, 20]])
@pytest.mark.parametrize("mxfp4", [False, True])
def test_what_is_not_seen_has_no_part(M, mxfp4, queries):
    """NaN and infinities in rows behind a sequence's last, in the pages of nobody, before a window
    and, for all but the queries behind them, in values that later queries see."""
    lens = [100, 90]

    def poison(pages, table):
        used = np.zeros(pages.shape[0] * 16, bool)
        for b, n in enumerate(lens):
            for j in range(n):
                used[table[b, j // 16] * 16 + j % 16] = True
        for b in range(2):  # the last but one key: the last query sees it alone
            j = lens[b] - 2
            used[table[b, j // 16] * 16 + j % 16] = False
        for page, row in np.argwhere(~used.reshape(-1, 16)):
            if pages.mxfp4:
                pages.ks[page, :, row] = pages.vs[page, :, row] = 255 if row % 2 else 254
            else:
                pages.k[page, :, row] = pages.v[page, :, row] = 0x7FC0 if row % 2 else 0xFF80

    run(M, lens, queries, mxfp4=mxfp4, edit=poison)
    # a window that the poisoned key is before for the last query
    if queries:
        run(M, lens, queries, mxfp4=mxfp4, edit=poison, window=1)


def test_pages_that_do_not_exist_hide_their_keys(M):
    def lose(pages, table):
        table[0, 2], table[0, 5] = -1, pages.shape[0]
        table[1, :] = 2 ** 31 - 1

    for queries in (None, [3, 4], [80, 30]):
        run(M, [120, 40], queries, edit=lose)
        run(M, [120, 40], queries, edit=lose, mxfp4=False, sinks=True)


def test_scores_of_any_size(M):
    """Scores of hundreds (a softmax of one key), and of both signs across steps and splits."""
    run(M, [300, 1500], heads=4, kv_heads=1, scale=3.0)
    run(M, [300, 1500], [70, 40], heads=4, kv_heads=1, scale=3.0, mxfp4=False)


def test_strides_streams_and_graphs(M):
    import torch

    rng = np.random.default_rng(11)
    lens = [40, 700, 3]
    table, n = K.page_tables(rng, lens, 32)
    pages = K.Pages(rng, n, 2, 32, 64, True)
    cache, table, lens = pages.device(M), X.dev(table), X.dev(np.array(lens, np.int32))
    for tokens, offsets in ((3, None), (50, [0, 30, 49, 50])):
        wide, _ = K.values_of(rng, (tokens, 8 * 64 * 3), False)
        q = wide[:, 8 * 64:16 * 64].view(tokens, 8, 64)
        how = dict(scale=0.2, q_offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        want = M.kv_attention(q.contiguous(), cache, table, lens, **how)
        out = torch.zeros(8, tokens, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
        M.kv_attention(q, cache, table, lens, out=out, **how)
        assert torch.equal(out, want)
        # a wide table
        big = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
        big[:, 5:5 + table.shape[1]] = table
        assert torch.equal(M.kv_attention(q, cache, big[:, 5:5 + table.shape[1]], lens, **how), want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        got = M.kv_attention(q, cache, table, lens, stream=side, **how)
        side.synchronize()
        assert torch.equal(got, want)


def test_no_pages_and_no_keys(M):
    import torch

    q = torch.ones(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    lens = torch.tensor([5, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for mxfp4 in (False, True):
        for pages, table in ((0, torch.zeros(3, 4, dtype=torch.int32, device="cuda")),
                             (2, torch.zeros(3, 0, dtype=torch.int32, device="cuda")),
                             (2, torch.full((3, 4), 2, dtype=torch.int32, device="cuda"))):
            cache = M.KVCache.zeros(pages, 2, 16, 64, mxfp4=mxfp4)
            for offsets in (None, torch.tensor([0, 1, 1, 3], dtype=torch.int32, device="cuda")):
                out, lse = M.kv_attention(q, cache, table, lens, scale=1.0, q_offsets=offsets, return_lse=True)
                assert (out == 0).all() and torch.isneginf(lse).all()


def test_lengths_and_offsets_that_do_not_fit(M):
    """A length past the table, or below zero; offsets that do not ascend or leave the tokens."""
    import torch

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    cache = M.KVCache.zeros(4, 2, 16, 64)
    cache.v.fill_(3)
    q = torch.ones(6, 4, 64, device="cuda", dtype=torch.bfloat16)
    table = i32([0, 1], [2, 3], [1, 2])
    out, lse = M.kv_attention(q[:3], cache, table, i32(1000, -5, 32), scale=1.0, return_lse=True)
    assert (out[0] == 3).all() and (out[1] == 0).all() and torch.allclose(lse[0], lse[2])
    for bad in (i32(0, 5, 2, 6), i32(-1, 2, 4, 6), i32(0, 2, 4, 7), i32(2 ** 31 - 1, -2 ** 31, 0, 3)):
        out = M.kv_attention(q, cache, table, i32(32, 32, 32), scale=1.0, q_offsets=bad, out=torch.full_like(q, 7))
        assert ((out == 3) | (out == 7)).all()
    out = M.kv_attention(q, cache, table, i32(32, 32, 32), scale=1.0, q_offsets=i32(0, 5, 2, 6), out=torch.full_like(q, 7))
    assert (out[:5] == 3).all()


def test_refusals(M):
    import torch

    cache = M.KVCache.zeros(4, 2, 16, 64, mxfp4=True)
    q = torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), i32(1, 2, 3)
    call = lambda q=q, cache=cache, table=table, lens=lens, scale=1.0, **kw: M.kv_attention(q, cache, table, lens, scale=scale, **kw)
    assert call().shape == q.shape
    off = torch.zeros(3 * 4 * 64 + 8, device="cuda", dtype=torch.bfloat16)
    bad = [
        lambda: call(q=q.float()), lambda: call(q=q[..., :32]), lambda: call(q=q[:, :3]), lambda: call(q=q[:2]),
        lambda: call(q=q.transpose(1, 2)), lambda: call(q=q.cpu()), lambda: call(table=table.long()), lambda: call(table=table[0]),
        lambda: call(lens=lens[:2]), lambda: call(lens=lens.long()), lambda: call(q_offsets=i32(0, 1, 2)),
        lambda: call(sinks=torch.zeros(3, device="cuda")), lambda: call(sinks=torch.zeros(4, device="cuda", dtype=torch.bfloat16)),
        lambda: call(scale=0.0), lambda: call(scale=float("nan")), lambda: call(scale=-1.0), lambda: call(window=-1),
        lambda: call(max_kv_len=-1), lambda: call(out=torch.zeros(3, 4, 32, device="cuda")),
        lambda: call(out=torch.zeros(3, 4, 64, device="cuda", dtype=torch.float16)),
        lambda: call(out=q[:1].expand(3, 4, 64)), lambda: call(q=off[1:1 + 768].view(3, 4, 64)),
        lambda: call(out=off[4:4 + 768].view(3, 4, 64)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((M.MRError, TypeError, ValueError)):
            f()
            print("accepted", i)
    assert M.kv_attention(q[:0], cache, table[:0], lens[:0], scale=1.0).shape == (0, 4, 64)
