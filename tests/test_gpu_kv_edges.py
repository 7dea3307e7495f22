"""Ends of the softmax of attention over a paged cache, in every form (whole and in parts, one
query and many, both joins): sinks of any f32, keys whose scores are all -inf, and infinite
values of keys whose probability is less than f32 holds.  Tolerances as in
test_gpu_kv_attention.py."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu
NAN, PLUS, MINUS = 0x7FC0, 0x7F80, 0xFF80  # bf16


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


# lengths, queries (None: one each, no offsets), heads, kv_heads: which form and join each takes is
# what tests/test_routes_kv_edges.py asks
FORMS = {
    "one": ([77, 0, 200], None, 8, 2),
    "one in parts": ([3000, 0, 700], None, 8, 2),
    "few": ([77, 9, 40], [3, 6, 0], 8, 2),
    "few in parts": ([3000, 0, 700], [7, 2, 9], 8, 2),
    "many": ([120, 130], [70, 60], 8, 2),
    "many in parts": ([900, 20, 0], [55, 17, 9], 8, 2),
    "many rows joined": ([900, 0, 300], [200, 20, 62], 8, 2),
}


def case(form, dim, mxfp4, seed=0):
    lens, queries, heads, kv_heads = FORMS[form]
    rng = np.random.default_rng([len(form), dim, mxfp4, seed])
    table, n = K.page_tables(rng, lens, 32)
    pages = K.Pages(rng, n, kv_heads, 32, dim, mxfp4)
    offsets = None if queries is None else np.cumsum([0] + list(queries)).astype(np.int32)
    T = len(lens) if queries is None else int(offsets[-1])
    q64 = X.from_bf16(X.to_bf16((1.5 * rng.standard_normal((T, heads, dim))).astype(np.float32))).astype(np.float64)
    return rng, table, pages, lens, offsets, q64


def attend(M, q64, pages, table, lens, offsets, scale, sinks=None, f32=True):
    """(out, lse) as 64-bit arrays."""
    import torch

    out, lse = M.kv_attention(X.dev(X.to_bf16(q64.astype(np.float32))), pages.device(M), X.dev(table),
                              X.dev(np.array(lens, np.int32)), scale=scale, sinks=None if sinks is None else X.dev(sinks),
                              q_offsets=None if offsets is None else X.dev(offsets), return_lse=True,
                              out_dtype=torch.float32 if f32 else torch.bfloat16)
    return X.host(out), X.host(lse)


def keys_seen(lens, offsets, tokens):
    """Of each token: [first, last) of its sequence's keys, and the sequence."""
    owner = np.arange(tokens) if offsets is None else np.searchsorted(offsets, np.arange(tokens), side="right") - 1
    end = np.arange(tokens) + 1 if offsets is None else offsets[owner + 1]
    return owner, np.maximum(np.array(lens)[owner] - (end - 1 - np.arange(tokens)), 0)


def compare(got, lse, want, lse64, weight, terms, dim, longest, f32):
    score = (dim + 2) * K.MFMA * terms[..., None]
    tol = weight * (X.BF16_ROUND + 2 * score + (longest + 8) * K.MFMA) + (X.F32_ROUND if f32 else X.BF16_ROUND) * np.abs(want) + 1e-37
    assert np.array_equal(np.isnan(got), np.isnan(want)), np.argwhere(np.isnan(got) != np.isnan(want))[:3]
    with np.errstate(invalid="ignore"):
        over = np.where(np.isnan(want) | (got == want), 0, np.abs(got - want) - tol)
        assert (over <= 0).all(), np.argwhere(over > 0)[:3]
        off = np.abs(lse - lse64) > score[..., 0] + 2.0 ** -21 * (1 + np.abs(lse64)) + longest * K.MFMA
    assert np.array_equal(np.isnan(lse), np.isnan(lse64)), np.argwhere(np.isnan(lse) != np.isnan(lse64))[:3]
    assert np.array_equal(lse[np.isinf(lse64)], lse64[np.isinf(lse64)])
    assert not (off & np.isfinite(lse64)).any(), np.argwhere(off & np.isfinite(lse64))[:3]


SINKS = np.array([3.4028235e38, -3.4028235e38, 3e38, np.nan, -np.inf, np.inf, 40.0, -40.0], np.float32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("mxfp4,dim", [(True, 128), (False, 64), (True, 256)])
@pytest.mark.parametrize("form", FORMS)
def test_sinks_of_any_size(M, form, dim, mxfp4, f32):
    """The largest and the least f32 ("no sink" of a mask's convention), both infinities, NaN.  A query
    without keys gets zeros and its sink as lse."""
    _, table, pages, lens, offsets, q64 = case(form, dim, mxfp4)
    scale = dim ** -0.5
    with np.errstate(invalid="ignore"):
        want, lse64, weight, terms = K.attention(q64, *pages.values(), table, lens, offsets, scale, 0, SINKS.astype(np.float64))
    none = keys_seen(lens, offsets, len(q64))[1] == 0
    want[none], lse64[none], weight[none] = 0, SINKS, 0
    got, lse = attend(M, q64, pages, table, lens, offsets, scale, SINKS, f32)
    compare(got, lse, want, lse64, weight, terms, dim, max(lens), f32)


@pytest.mark.parametrize("mxfp4,dim", [(True, 128), (False, 64), (False, 256)])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("form", FORMS)
def test_scores_that_are_all_minus_infinity(M, form, sinks, dim, mxfp4):
    """As without keys, also where the values are infinite; other heads and sequences have none of it."""
    _, table, pages, lens, offsets, q64 = case(form, dim, mxfp4)
    q64 = X.from_bf16(X.to_bf16((np.abs(q64) + 0.5).astype(np.float32))).astype(np.float64)
    hidden = table[0, :-(-lens[0] // 32)]  # the first sequence's keys, of key head 0
    if mxfp4:
        pages.k[hidden, 0, :, :4], pages.ks[hidden, 0, :, 0] = 0xFFFFFFFF, 254  # -6 2^127
        pages.v[hidden[-1:], 0, :, 4:8], pages.vs[hidden[-1:], 0, :, 1] = 0x77777777, 254
    else:
        pages.k[hidden, 0, :, 3] = MINUS
        pages.v[hidden[-1:], 0, :, 9] = PLUS
    s = np.linspace(-3, 3, 8).astype(np.float32) if sinks else None
    scale = dim ** -0.5
    with np.errstate(invalid="ignore"):
        want, lse64, weight, terms = K.attention(q64, *pages.values(), table, lens, offsets, scale, 0,
                                                 None if s is None else s.astype(np.float64))
    owner, seen = keys_seen(lens, offsets, len(q64))
    for t in range(len(q64)):
        if owner[t] == 0 or seen[t] == 0:
            heads = slice(0, 4) if seen[t] else slice(0, 8)
            want[t, heads], weight[t, heads], terms[t, heads] = 0, 0, 0
            lse64[t, heads] = -np.inf if s is None else s[heads]
    got, lse = attend(M, q64, pages, table, lens, offsets, scale, s)
    compare(got, lse, want, lse64, weight, terms, dim, max(lens), True)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("mxfp4,dim", [(True, 64), (True, 128), (False, 128), (True, 256), (False, 96)])
@pytest.mark.parametrize("sink", [None, 2000.0])
@pytest.mark.parametrize("form", FORMS)
def test_infinite_values_of_any_probability(M, form, sink, dim, mxfp4, f32):
    """Scores of +-150 and more, so that most probabilities are less than f32 holds (with the sink: all).
    Infinite values reach every query that sees them, whichever tile or part they are in."""
    rng, table, pages, lens, offsets, q64 = case(form, dim, mxfp4, 1)
    scale, kv_heads = 3.0, pages.shape[1]
    cols = 32 if mxfp4 else 1
    odd = {}  # (sequence, key, key head) -> {dim: value}
    for b, n in enumerate(lens):
        for j in {0, 1, n // 2, n - 1, n - 2, *rng.integers(0, max(n, 1), 6).tolist()}:
            if not 0 <= j < n:
                continue
            page, row, h = table[b, j // 32], j % 32, int(rng.integers(kv_heads))
            block, value = int(rng.integers(dim // cols)), [np.inf, -np.inf, np.nan][int(rng.choice(3, p=[0.45, 0.45, 0.1]))]
            odd[b, j, h] = {d: value for d in range(block * cols, (block + 1) * cols)}
            if not mxfp4:
                pages.v[page, h, row, block] = {np.inf: PLUS, -np.inf: MINUS}.get(value, NAN)
            elif np.isnan(value):
                pages.vs[page, h, row, block] = 255
            else:
                pages.vs[page, h, row, block] = 254
                pages.v[page, h, row, 4 * block:4 * block + 4] = 0x77777777 if value > 0 else 0xFFFFFFFF
    s = None if sink is None else np.full(q64.shape[1], sink, np.float32)
    k64, v64 = pages.values()
    want, lse64, weight, terms = K.attention(q64, k64, np.where(np.isfinite(v64), v64, 0), table, lens, offsets, scale, 0,
                                             None if s is None else s.astype(np.float64))
    owner, seen = keys_seen(lens, offsets, len(q64))
    none = seen == 0
    want[none], weight[none] = 0, 0
    lse64[none] = -np.inf if s is None else sink
    with np.errstate(invalid="ignore"):
        for (b, j, h), dims in odd.items():
            rows = np.flatnonzero((owner == b) & (seen > j))
            for d, value in dims.items():
                want[rows[:, None], np.arange(4 * h, 4 * h + 4)[None], d] += value
    got, lse = attend(M, q64, pages, table, lens, offsets, scale, s, f32)
    compare(got, lse, want, lse64, weight, terms, dim, max(lens), f32)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("mxfp4", [False, True])
def test_values_that_are_all_nan(M, form, mxfp4):
    _, table, pages, lens, offsets, q64 = case(form, 128, mxfp4)
    if mxfp4:
        pages.vs[:] = 255
    else:
        pages.v[:] = NAN
    got, lse = attend(M, q64, pages, table, lens, offsets, 0.1)
    none = keys_seen(lens, offsets, len(q64))[1] == 0
    assert np.isnan(got[~none]).all() and (got[none] == 0).all() and np.array_equal(np.isneginf(lse).all(1), none)
