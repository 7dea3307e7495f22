"""Norms of query and key heads with the rotation, and their gradients, on the GPU
against 64 bits.

Tolerances (u = 2^-24): the sum of squares is a chain of 8 and up to 6 steps
between lanes, halved by the root, so 1 / norm is off by at most 10 u, the
normalised and weighted value by 12 u, and a rotation adds a product and a sum: 14 u
of the magnitudes it adds.  Gradients: kv_inputs.norm_backward has the terms of dx
with 15 and 54 roundings; a term of dw has 14, its sum as many as the longest chain of
sums (rows of a lane, 6 + 4 of a workgroup, 64 + 16 partial rows).  Outputs are rounded
once to their type."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu
EPS = 1e-6

# tokens, heads, kv_heads, dim, rotated columns, first of them, halves
SHAPES = [
    (1, 1, 1, 1, 0, 0, False), (1, 32, 4, 128, 128, 0, True), (3, 2, 1, 2, 2, 0, False), (5, 4, 2, 64, 64, 0, False),
    (17, 3, 1, 96, 64, 32, False), (17, 3, 1, 96, 64, 32, True), (9, 5, 0, 512, 64, 448, False), (33, 8, 2, 256, 128, 0, True),
    (7, 2, 2, 33, 14, 3, True), (7, 2, 2, 33, 14, 3, False), (6, 1, 3, 72, 40, 16, True), (6, 1, 3, 72, 40, 16, False),
    (257, 6, 2, 128, 32, 96, True), (11, 7, 5, 8, 8, 0, False), (4, 2, 1, 500, 500, 0, True), (700, 16, 2, 40, 24, 8, False),
]


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def inputs(shape, f32, weights="both"):
    T, H, G, D, rope, col0, halves = shape
    rng = np.random.default_rng([T, H, D, rope, f32])
    q, q64 = K.values_of(rng, (T, H, D), f32, 2.0)
    k, k64 = K.values_of(rng, (T, G, D), f32, 0.1)
    w32 = weights == "f32"
    wq, wq64 = K.values_of(rng, (D,), w32)
    wk, wk64 = K.values_of(rng, (D,), w32)
    cos, sin = K.tables(rng, T + 5, rope // 2)
    positions = rng.integers(0, T + 5, T).astype(np.int32)
    how = dict(eps=EPS, col0=col0, halves=halves)
    if weights == "none":
        wq64 = wk64 = np.ones(D)
    else:
        how["q_weight"] = wq
        if G:
            how["k_weight"] = wk
    if rope:
        how.update(cos_t=X.dev(cos), sin_t=X.dev(sin), positions=X.dev(positions))
    return rng, (q, q64, wq64), (k, k64, wk64) if G else None, (cos[positions], sin[positions]), how


def check(got, want, bound, f32, tag):
    err = np.abs(X.host(got) - want)
    tol = bound + (X.F32_ROUND if f32 else X.BF16_ROUND) * np.abs(want) + 1e-37
    worst = np.unravel_index(np.argmax(err - tol), err.shape) if err.size else None
    assert (err <= tol).all(), (tag, worst, err[worst], tol[worst])


@pytest.mark.parametrize("f32,out_f32,weights", [(False, False, "both"), (True, True, "f32"), (False, True, "none"),
                                                 (True, False, "both")])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(M, shape, f32, out_f32, weights):
    import torch

    _, q, k, (cos, sin), how = inputs(shape, f32, weights)
    col0, halves = shape[5:]
    out = M.head_norm_rope(q[0], k and k[0], out_dtype=torch.float32 if out_f32 else torch.bfloat16, **how)
    for (x, x64, w), y, tag in zip((q, k), (out,) if k is None else out, "qk"):
        n = K.norm(x64, w, EPS)
        check(y, K.turn(n, cos, sin, col0, halves), 14 * K.U * K.spread(n, cos, sin, col0, halves), out_f32, tag)


@pytest.mark.parametrize("f32,weights", [(False, "both"), (True, "f32"), (True, "none")])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(M, shape, f32, weights):
    rng, q, k, (cos, sin), how = inputs(shape, f32, weights)
    T, col0, halves = shape[0], *shape[5:]
    d = [K.values_of(rng, t[1].shape, f32) for t in (q, k) if t]
    got = M.head_norm_rope_backward(d[0][0], q[0], *((d[1][0], k[0]) if k else ()), **how)
    got = [got] if k is None else [(got[0], got[2]), (got[1], got[3])]
    for (x, x64, w), (_, dy), (dx, dw), tag in zip((q, k), d, got, "qk"):
        want, want_w, bound, total = K.norm_backward(dy, x64, w, EPS, cos, sin, col0, halves)
        check(dx, want, K.U * bound, f32, tag)
        if weights == "none":
            assert dw is None
            continue
        chain = 14 + T * x64.shape[1] // 16 + 1 + 90
        assert (np.abs(X.host(dw) - want_w) <= chain * K.U * total + K.U * np.abs(want_w)).all(), tag


def test_gradients_against_differences(M):
    """Central differences of sum(dy * y) in 64 bits (the function is smooth: an error of step^2)."""
    shape = (3, 2, 1, 24, 16, 4, True)
    rng, q, k, (cos, sin), how = inputs(shape, True, "f32")
    d = [K.values_of(rng, t[1].shape, True) for t in (q, k)]
    got = M.head_norm_rope_backward(d[0][0], q[0], d[1][0], k[0], **how)
    step = 1e-5
    for i, (x, x64, w) in enumerate((q, k)):
        f = lambda x, w: (d[i][1] * K.turn(K.norm(x, w, EPS), cos, sin, 4, True)).sum()
        for which, g in ((0, got[i]), (1, got[2 + i])):
            at = [x64, w]
            g = X.host(g).reshape(-1)
            for j in range(0, g.size, 5):
                e = np.zeros(at[which].size)
                # a step small beside the row's size
                e[j] = step * (np.abs(x64).max() if which == 0 else 1)
                e = e.reshape(at[which].shape)
                hi, lo = [a.copy() for a in at], [a.copy() for a in at]
                hi[which], lo[which] = hi[which] + e, lo[which] - e
                slope = (f(*hi) - f(*lo)) / (2 * e.sum())
                # f32 roundings (60 of terms like the largest gradients) and the difference's own error
                assert abs(g[j] - slope) <= 60 * K.U * np.abs(g).max() + 1e-6 * np.abs(g).max(), (i, which, j)


def test_sums_of_many_rows_do_not_depend_on_the_run(M):
    import torch

    shape = (4099, 8, 2, 128, 128, 0, True)
    _, q, k, _, how = inputs(shape, False)
    runs = [M.head_norm_rope_backward(q[0], q[0], k[0], k[0], **how) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_strides_in_place_and_no_tokens(M):
    import torch

    rng = np.random.default_rng(5)
    T, H, G, D = 9, 4, 2, 64
    # queries, keys and values of a projection in one row
    fused, f64 = K.values_of(rng, (T, (H + 2 * G) * D), False)
    q, k = fused[:, :H * D].view(T, H, D), fused[:, H * D:(H + G) * D].view(T, G, D)
    cos, sin = K.tables(rng, T, D // 2)
    how = dict(cos_t=X.dev(cos), sin_t=X.dev(sin))
    a, b = M.head_norm_rope(q.contiguous(), k.contiguous(), **how)
    before = fused.clone()
    # heads first in memory, and rows off a 16-byte boundary
    y = torch.full((H, T, D), 7.0, device="cuda", dtype=torch.bfloat16)
    wide = torch.full((T, G, D + 3), 7.0, device="cuda", dtype=torch.bfloat16)
    M.head_norm_rope(q, k, q_out=y.transpose(0, 1), k_out=wide[:, :, 1:D + 1], **how)
    assert torch.equal(y.transpose(0, 1), a) and torch.equal(wide[:, :, 1:D + 1], b)
    assert (wide[:, :, 0] == 7).all() and (wide[:, :, D + 1:] == 7).all()
    # a repeated row (stride 0) may be read
    one = q[:1].expand(T, H, D)
    assert torch.equal(M.head_norm_rope(one, **how), M.head_norm_rope(one.contiguous(), **how))
    M.head_norm_rope(q, k, q_out=q, k_out=k, **how)
    assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(fused[:, (H + G) * D:], before[:, (H + G) * D:])
    w = torch.ones(D, device="cuda")
    empty = torch.empty(0, H, D, device="cuda")
    assert M.head_norm_rope(empty).shape == (0, H, D)
    dx, dw = M.head_norm_rope_backward(empty, empty, q_weight=w)
    assert dx.shape == (0, H, D) and (dw == 0).all()


def test_positions_outside_the_tables_and_rows_of_zeros(M):
    import torch

    T, H, D = 4, 2, 32
    x = torch.ones(T, H, D, device="cuda")
    x[3] = 0
    cos = torch.ones(6, 8, device="cuda")
    y = M.head_norm_rope(x, cos_t=cos, sin_t=cos, positions=torch.tensor([0, 6, -1, 5], dtype=torch.int32, device="cuda"), col0=4)
    assert torch.isnan(y[1:3, :, 4:20]).all() and torch.isfinite(y[1:3, :, :4]).all() and torch.isfinite(y[1:3, :, 20:]).all()
    assert torch.isfinite(y[0]).all() and (y[3] == 0).all()
    # a NaN stays in its head
    x[0, 1, 5] = float("nan")
    y = M.head_norm_rope(x)
    assert torch.isnan(y[0, 1]).all() and torch.isfinite(y[0, 0]).all() and torch.isfinite(y[1:]).all()


def test_refusals(M):
    import torch

    q = torch.zeros(4, 2, 32, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(4, 8, device="cuda")
    bad = [
        lambda: M.head_norm_rope(q.cpu()), lambda: M.head_norm_rope(q.half()), lambda: M.head_norm_rope(q[0]),
        lambda: M.head_norm_rope(q.transpose(1, 2)), lambda: M.head_norm_rope(q, q[:3]), lambda: M.head_norm_rope(q, q.float()),
        lambda: M.head_norm_rope(q, q_weight=torch.ones(31, device="cuda")),
        lambda: M.head_norm_rope(q, k_weight=torch.ones(32, device="cuda")),
        lambda: M.head_norm_rope(q, q_weight=torch.ones(32, device="cuda", dtype=torch.float16)),
        lambda: M.head_norm_rope(q, cos_t=table), lambda: M.head_norm_rope(q, cos_t=table, sin_t=table[:3]),
        lambda: M.head_norm_rope(q, cos_t=table[:3], sin_t=table[:3]),
        lambda: M.head_norm_rope(q, cos_t=table, sin_t=table, col0=17),
        lambda: M.head_norm_rope(q, cos_t=table, sin_t=table, positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: M.head_norm_rope(q, cos_t=table, sin_t=table, positions=torch.zeros(4, dtype=torch.int64, device="cuda")),
        lambda: M.head_norm_rope(q, eps=float("nan")), lambda: M.head_norm_rope(q, eps=-1.0),
        lambda: M.head_norm_rope(q, q_out=q[:1].expand(4, 2, 32)), lambda: M.head_norm_rope(q, q_out=q.float(), out_dtype=q.dtype),
        lambda: M.head_norm_rope(torch.zeros(1, 1, 513, device="cuda")),
        lambda: M.head_norm_rope_backward(q, q, q), lambda: M.head_norm_rope_backward(q.float(), q),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((M.MRError, TypeError, ValueError)):
            call()
            print("accepted", i)
