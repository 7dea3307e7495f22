"""Products with MXFP4 weights on the GPU, of one matrix and of experts' rows.

Two kinds of inputs.  Whole numbers and halves: every product is a multiple of
1/8 and every partial sum is below 2^24 / 8, so any order of f32 sums is exact
and the outputs must be too.  Normal values: a sum of n products rounds at most
n times, each time by at most 2^-24 of a partial sum, which is at most the sum
of the magnitudes (n = K, 3 K for f32 activations, whose three parts are
multiplied one by one); the output rounds once more to its type."""
import numpy as np
import pytest

import mxfp4_inputs as X

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f32", "mxfp4"]


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def whole(rng, kind, rows, cols):
    """x of small whole numbers (MXFP4: halves too): operand and 64-bit values."""
    if kind == "mxfp4":
        packed, scales = X.matrix(rng, rows, cols, lo=126, hi=129)
        return (packed, scales), X.values(packed, scales)
    x = rng.integers(-8, 9, (rows, cols)).astype(np.float32)
    return (x if kind == "f32" else X.to_bf16(x)), x.astype(np.float64)


def normal(rng, kind, rows, cols):
    if kind == "mxfp4":
        packed, scales = X.matrix(rng, rows, cols)
        return (packed, scales), X.values(packed, scales)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x = x if kind == "f32" else X.to_bf16(x)
    return x, (x if kind == "f32" else X.from_bf16(x)).astype(np.float64)


def operand(M, x):
    return M.MXFP4Weights(X.dev(x[0]), X.dev(x[1])) if isinstance(x, tuple) else X.dev(x)


def weights(M, rng, rows, cols, lead=(), **kw):
    packed, scales = X.matrix(rng, rows, cols, lead, **kw)
    return M.MXFP4Weights(X.dev(packed), X.dev(scales)), X.values(packed, scales)


def bound(kind, x64, w64, y64, out_round):
    n = w64.shape[-1] * (3 if kind == "f32" else 1)
    return (n * X.F32_ROUND * (np.abs(x64) @ np.abs(w64).T) + out_round * np.abs(y64)) * 1.01


TOKENS = [1, 2, 3, 4, 5, 8, 16, 17, 33, 64, 65, 130, 257, 300]
SHAPES = [(1, 32), (7, 64), (16, 96), (33, 128), (96, 160), (257, 1056), (40, 2080), (512, 512), (300, 4096)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("out,inp", SHAPES)
def test_whole_numbers_are_exact(M, out, inp, kind):
    import torch

    rng = np.random.default_rng(out + inp)
    w, w64 = weights(M, rng, out, inp, lo=126, hi=129)
    x, x64 = whole(rng, kind, max(TOKENS), inp)
    for tokens in TOKENS:
        part = (x[0][:tokens], x[1][:tokens]) if kind == "mxfp4" else x[:tokens]
        print(f"mm {kind} {tokens} x {out} x {inp}", flush=True)
        y = M.mxfp4_mm(operand(M, part), w, out_dtype=torch.float32)
        want = x64[:tokens] @ w64.T
        assert np.abs(want).max() < 2 ** 21
        assert np.array_equal(X.host(y), want), (tokens, np.abs(X.host(y) - want).max())
        yb = M.mxfp4_mm(operand(M, part), w, out_dtype=torch.bfloat16)
        assert torch.equal(yb, y.bfloat16())


# token and output counts on both sides of every change of kernel or tile (a few
# outputs to most of the GPU's workgroups, one token to tiles of 256), K with and
# without a remainder
WIDE = [(1, 300, 544), (2, 300, 4128), (20, 300, 288), (10, 4104, 288), (40, 2056, 544), (100, 2056, 160), (100, 4000, 288),
        (100, 4104, 256), (40, 16392, 96), (10, 33000, 96), (100, 8200, 2080), (20, 300, 4128), (100, 16392, 288),
        (200, 16392, 288), (300, 16392, 512), (600, 16392, 256), (600, 16385, 288), (700, 16390, 32), (1100, 8190, 416),
        (1000, 16384, 512), (1000, 16300, 288), (100, 8200, 544), (20, 8200, 96),
        (100, 2056, 2080), (300, 2056, 96), (400, 2056, 4128), (100, 264, 544)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,out,inp", WIDE)
def test_whole_numbers_are_exact_in_every_kernel(M, tokens, out, inp, kind):
    import torch

    rng = np.random.default_rng(tokens + out)
    w, w64 = weights(M, rng, out, inp, lo=126, hi=129)
    x, x64 = whole(rng, kind, tokens, inp)
    want = (x64.astype(np.float32) @ w64.astype(np.float32).T).astype(np.float64)  # exact: see above
    assert np.abs(want).max() < 2 ** 21
    y = M.mxfp4_mm(operand(M, x), w, out_dtype=torch.float32)
    assert np.array_equal(X.host(y), want), np.abs(X.host(y) - want).max()
    assert torch.equal(M.mxfp4_mm(operand(M, x), w, out_dtype=torch.bfloat16), y.bfloat16())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,out,inp", [(1, 1536, 7168), (13, 576, 7168), (37, 1536, 1536), (200, 768, 2048),
                                            (1000, 512, 512), (300, 2048, 7168)])
def test_normal_values(M, tokens, out, inp, kind):
    import torch

    rng = np.random.default_rng(tokens)
    w, w64 = weights(M, rng, out, inp, std=inp ** -0.5)
    x, x64 = normal(rng, kind, tokens, inp)
    want = x64 @ w64.T
    for dt, r in ((torch.bfloat16, X.BF16_ROUND), (torch.float32, X.F32_ROUND)):
        got = X.host(M.mxfp4_mm(operand(M, x), w, out_dtype=dt))
        assert (np.abs(got - want) <= bound(kind, x64, w64, want, r)).all(), np.abs(got - want).max()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 3, 40, 300])
@pytest.mark.parametrize("inp", [32, 96, 160, 608])
def test_a_nan_block_stays_in_its_row(M, inp, tokens, kind):
    # every second weight row ends in a NaN block and starts with one, so that
    # the bytes next to the other rows' are NaN scales
    rng = np.random.default_rng(inp)
    packed, scales = X.matrix(rng, 37, inp, lo=126, hi=129)
    scales[1::2, -1] = scales[1::2, 0] = 255
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    x, x64 = whole(rng, kind, tokens, inp)
    if kind == "mxfp4":
        x[1][1::2, 0] = x[1][1::2, -1] = 255
        x64 = X.values(*x)
    got = X.host(M.mxfp4_mm(operand(M, x), w, out_dtype=__import__("torch").float32))
    want = np.where(np.isnan(x64).any(1)[:, None], np.nan, 0) + np.nan_to_num(x64) @ X.values(packed, scales)[::2].T
    assert np.isnan(got[:, 1::2]).all()
    assert np.array_equal(got[:, ::2], want, equal_nan=True)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [2, 70, 300])
def test_activations_that_are_not_finite(M, tokens, kind):
    import torch

    rng = np.random.default_rng(tokens)
    packed, scales = X.matrix(rng, 70, 96, lo=126, hi=129)
    packed |= np.uint32(0x22222222)  # no weight is zero
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    x, x64 = whole(rng, kind, tokens, 96)
    x64 = x64.copy()
    x64[0, 40], x64[1, 95] = np.inf, np.nan
    x = x64.astype(np.float32) if kind == "f32" else X.to_bf16(x64)
    got = X.host(M.mxfp4_mm(operand(M, x), w, out_dtype=torch.float32))
    w64 = X.values(packed, scales)
    assert np.array_equal(got[0], np.sign(w64[:, 40]) * np.inf)
    assert np.isnan(got[1]).all()
    assert np.array_equal(got[2:], x64[2:] @ w64.T)


def test_f32_activations_are_taken_whole(M):
    # 24 significant bits, one per row, against weights of one
    import torch

    rng = np.random.default_rng(1)
    x = np.zeros((64, 96), np.float32)
    x[np.arange(64), rng.integers(0, 96, 64)] = rng.standard_normal(64).astype(np.float32) * np.exp2(rng.integers(-100, 100, 64))
    x[0] = 0
    x[0, 5] = np.float32(3.4028234e38)
    w = M.MXFP4Weights(X.dev(np.full((20, 12), 0x22222222, np.uint32)), X.dev(np.full((20, 3), 127, np.uint8)))
    got = X.host(M.mxfp4_mm(X.dev(x), w, out_dtype=torch.float32))
    assert np.array_equal(got, np.repeat(x.sum(1, dtype=np.float64)[:, None], 20, 1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_ends_of_the_scale_range(M, tokens, kind):
    # weights near 2^-127 against activations near 2^100 and the other way
    # round: products in range, whatever the parts are
    import torch

    rng = np.random.default_rng(tokens)
    for wb, xb in ((0, 240), (2, 230), (240, 14)):
        packed, scales = X.matrix(rng, 33, 160, lo=wb, hi=wb + 2)
        w, w64 = M.MXFP4Weights(X.dev(packed), X.dev(scales)), X.values(packed, scales)
        if kind == "mxfp4":
            x = X.matrix(rng, tokens, 160, lo=xb, hi=xb + 2)
            x64 = X.values(*x)
        else:
            x64 = rng.integers(-8, 9, (tokens, 160)) * 2.0 ** (xb - 127)
            x = x64.astype(np.float32) if kind == "f32" else X.to_bf16(x64)
        got = X.host(M.mxfp4_mm(operand(M, x), w, out_dtype=torch.float32))
        assert np.array_equal(got, x64 @ w64.T)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_strides(M, kind):
    import ctypes as C
    import torch

    rng = np.random.default_rng(2)
    for tokens, out, inp in ((5, 33, 96), (300, 264, 160)):
        w, w64 = weights(M, rng, out, inp, lo=126, hi=129)
        x, x64 = whole(rng, kind, tokens, inp)
        buf = torch.full((tokens, inp + 16), float("nan"), dtype=torch.float32 if kind == "f32" else torch.bfloat16,
                         device="cuda")
        buf[:, 8:8 + inp] = X.dev(x)
        for dt in (torch.float32, torch.bfloat16):
            for start, width in ((0, out + 8), (3, out + 5)):
                y = torch.full((tokens, width), -77.0, dtype=dt, device="cuda")
                v, xv = y[:, start:start + out], buf[:, 8:8 + inp]
                M._check(M.load().mr_mxfp4_matmul(M._ptr(xv), M._dtype_code(xv.dtype), tokens, xv.stride(0),
                                                  C.byref(w.desc()), M._ptr(v), M._dtype_code(dt), width, M._stream(None)))
                want = torch.from_numpy(x64 @ w64.T).to(dt).double().numpy()
                assert np.array_equal(X.host(v), want)
                y[:, start:start + out] = -77
                assert (y == -77).all()


def test_vector_and_no_tokens(M):
    import torch

    rng = np.random.default_rng(3)
    w, w64 = weights(M, rng, 48, 64, lo=126, hi=129)
    x, x64 = whole(rng, "bf16", 1, 64)
    y = M.mxfp4_mm(X.dev(x)[0], w)
    assert y.shape == (48,) and y.dtype == torch.bfloat16
    assert M.mxfp4_mm(X.dev(x)[:0], w).shape == (0, 48)
    empty = M.mxfp4_quantize(X.dev(x)[:0])
    assert M.mxfp4_mm(empty, w).shape == (0, 48)


def test_offsets_past_32_bits(M):
    # weights of 2^32 values and 2^31 bytes, rows far from each other checked
    import torch

    rows, cols = 131073, 32768
    packed = torch.full((rows, cols // 8), 0x22222222, dtype=torch.int32, device="cuda")
    scales = torch.full((rows, cols // 32), 127, dtype=torch.uint8, device="cuda")
    at = [0, 1, 65535, 65536, 131071, 131072]
    for i, r in enumerate(at):
        scales[r] = 127 + i
    w = M.MXFP4Weights(packed, scales)
    x = torch.zeros(3, cols, device="cuda", dtype=torch.bfloat16)
    x[:, -1], x[1, 0] = 1, 2
    y = M.mxfp4_mm(x, w, out_dtype=torch.float32)
    for i, r in enumerate(at):
        assert y[:, r].tolist() == [2.0 ** i, 3 * 2.0 ** i, 2.0 ** i]
    assert int((y[0] == 1).sum()) == rows - len(at) + 1


EXPERTS = [(1, 1, 1, 7, 32), (1, 8, 128, 96, 256), (5, 2, 3, 33, 96), (40, 3, 9, 160, 160), (200, 8, 32, 264, 512),
           (700, 4, 5, 512, 288), (64, 6, 257, 48, 64), (1500, 2, 4, 300, 1024), (40, 4, 40, 136, 544), (90, 8, 60, 520, 288),
           (260, 8, 60, 264, 96), (300, 8, 60, 600, 544), (500, 8, 60, 392, 512), (500, 8, 60, 520, 288),
           (260, 8, 100, 700, 256), (260, 8, 100, 700, 288), (3, 2, 9, 48, 1024), (7, 4, 14, 40, 544),
           (100, 4, 150, 500, 160), (30, 4, 60, 340, 96)]


@pytest.mark.parametrize("ids", ["spread", "hot", "one", "dropped", "none", "twice"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,per_token,experts,out,inp", EXPERTS)
def test_experts_whole_numbers_are_exact(M, tokens, per_token, experts, out, inp, kind, ids):
    import torch

    rng = np.random.default_rng(tokens + inp)
    ids = X.ids_of(rng, tokens, per_token, experts, ids)
    offsets, pair, _ = X.order(ids, experts)
    o = M.expert_sort(X.dev(ids), experts)
    w, w64 = weights(M, rng, out, inp, (experts,), lo=126, hi=129)
    pairs, n = tokens * per_token, int(offsets[-1])
    for by_row in (False, True):
        x, x64 = whole(rng, kind, pairs if by_row else tokens, inp)
        want = np.full((pairs, out), -3.0)
        for e in range(experts):
            r = np.arange(offsets[e], offsets[e + 1])
            if r.size:
                want[r] = x64[r if by_row else pair[r] // per_token] @ w64[e].T
        for dt in (torch.float32, torch.bfloat16):
            print(f"experts {kind} {tokens} x {per_token} of {experts}, {out} x {inp}, by row {by_row}", flush=True)
            left = torch.full((pairs, out), -3.0, dtype=dt, device="cuda")
            y = M.mxfp4_expert_mm(operand(M, x), w, o, sorted_rows=by_row, out=left)
            assert np.array_equal(X.host(y), torch.from_numpy(want).to(dt).double().numpy()), (kind, by_row)


@pytest.mark.parametrize("kind", KINDS)
def test_experts_of_real_widths(M, kind):
    import torch

    rng = np.random.default_rng(7)
    tokens, per_token, experts, out, inp = 300, 8, 16, 768, 2048
    o = M.expert_sort(X.dev(X.ids_of(rng, tokens, per_token, experts, "hot")), experts)
    offsets, pair = o.offsets.tolist(), o.pair_of_row.cpu().numpy()
    w, w64 = weights(M, rng, out, inp, (experts,), std=inp ** -0.5)
    x, x64 = normal(rng, kind, tokens, inp)
    got = X.host(M.mxfp4_expert_mm(operand(M, x), w, o, out_dtype=torch.bfloat16))
    for e in range(experts):
        r = slice(offsets[e], offsets[e + 1])
        xe = x64[pair[r] // per_token]
        want = xe @ w64[e].T
        assert (np.abs(got[r] - want) <= bound(kind, xe, w64[e], want, X.BF16_ROUND)).all()


def test_a_layer_of_experts(M):
    """The run of a layer: ids sorted, both projections of each expert's rows
    (the first from the tokens, the second of rows in expert order, activations
    quantised on the way), results back to the tokens; each stage against 64
    bits on what the stage before it left."""
    import torch

    rng = np.random.default_rng(21)
    tokens, per_token, experts, hidden, inner = 150, 4, 12, 512, 256
    ids = X.ids_of(rng, tokens, per_token, experts, "dropped")
    x = torch.from_numpy(rng.standard_normal((tokens, hidden)).astype(np.float32)).cuda().bfloat16()
    router = torch.rand(tokens, per_token, device="cuda")
    up, up64 = weights(M, rng, 2 * inner, hidden, (experts,), std=hidden ** -0.5)
    down, down64 = weights(M, rng, hidden, inner, (experts,), std=inner ** -0.5)

    def layer(quantised):
        o = M.expert_sort(X.dev(ids), experts)
        h = M.mxfp4_expert_mm(M.mxfp4_quantize(x) if quantised else x, up, o, out_dtype=torch.bfloat16)
        n = int(o.offsets[-1])
        h[n:] = 0
        a = (torch.nn.functional.silu(h[:, :inner].float()) * h[:, inner:].float()).bfloat16()
        y = M.mxfp4_expert_mm(M.mxfp4_quantize(a) if quantised else a, down, o, sorted_rows=True, out_dtype=torch.bfloat16)
        return o, n, h, a, y, M.expert_combine(y, o, router)

    for quantised in (False, True):
        o, n, h, a, y, out = layer(quantised)
        offsets, pair = o.offsets.tolist(), o.pair_of_row.cpu().numpy()
        seen = lambda t: X.host(M.mxfp4_dequantize(M.mxfp4_quantize(t))) if quantised else X.host(t)
        x64, a64, kind = seen(x), seen(a), "mxfp4" if quantised else "bf16"
        for e in range(experts):
            r = slice(offsets[e], offsets[e + 1])
            for got, rows, w64 in ((h, x64[pair[r] // per_token], up64[e]), (y, a64[r], down64[e])):
                want = rows @ w64.T
                assert (np.abs(X.host(got[r]) - want) <= bound(kind, rows, w64, want, X.BF16_ROUND)).all()
        row = o.row_of_pair.cpu().numpy()
        terms = np.where((row >= 0)[..., None], X.host(router)[..., None] * X.host(y)[np.maximum(row, 0)], 0)
        tol = per_token * X.F32_ROUND * np.abs(terms).sum(1) + X.BF16_ROUND * np.abs(terms.sum(1))
        assert (np.abs(X.host(out) - terms.sum(1)) <= tol * 1.01).all()


def test_graph_replays_and_other_streams(M):
    import torch

    rng = np.random.default_rng(12)
    tokens, per_token, experts, out, inp = 90, 3, 7, 200, 160
    ids = X.dev(X.ids_of(rng, tokens, per_token, experts, "spread"))
    x = torch.randn(tokens, inp, device="cuda", dtype=torch.bfloat16)
    w, _ = weights(M, rng, out, inp, (experts,))
    one, _ = weights(M, rng, out, inp)
    left = torch.zeros(tokens * per_token, out, device="cuda", dtype=torch.bfloat16)

    def step(stream=None):
        q = M.mxfp4_quantize(x, stream=stream)
        o = M.expert_sort(ids, experts, stream=stream)
        y = M.mxfp4_expert_mm(q, w, o, out=left, stream=stream)
        return M.expert_combine(y, o, stream=stream), M.mxfp4_mm(x, one, stream=stream), M.mxfp4_mm(q, one, stream=stream)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = step(s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for kind in ("hot", "dropped", "one"):
        ids.copy_(X.dev(X.ids_of(rng, tokens, per_token, experts, kind)))
        x.copy_(torch.randn(tokens, inp, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
