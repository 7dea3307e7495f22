"""Tokens sorted by expert and back on the GPU: the order exactly, dispatched
rows bit for bit, sums and gradients against 64 bits.

Tolerances: combine sums K products with f32 fused multiply-adds (K roundings
of a partial sum that is at most the sum of |w y|) and rounds once to the
type; a weight's gradient sums dim products, in chains of at most
ceil(dim / 2048) * 8 + 8 roundings per thread and 10 between threads, each of a
partial sum at most sum |g y|; d_rows is one product (f32) and one rounding."""
import numpy as np
import pytest

import mxfp4_inputs as X

pytestmark = pytest.mark.gpu

KINDS = ["spread", "hot", "one", "dropped", "none", "twice"]


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def type_round(f32):
    return X.F32_ROUND if f32 else X.BF16_ROUND


def rows_of(rng, n, dim, f32):
    """(device tensor, the same in 64 bits)."""
    x = rng.standard_normal((n, dim)).astype(np.float32)
    x = x if f32 else X.to_bf16(x)
    return X.dev(x), (x if f32 else X.from_bf16(x)).astype(np.float64)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,per_token,experts", [
    (1, 1, 1), (1, 8, 128), (3, 2, 5), (64, 1, 2), (63, 7, 60), (512, 8, 128), (513, 8, 256), (1000, 6, 257),
    (4099, 3, 64), (2500, 5, 4096), (20000, 4, 700)])
def test_sort_is_the_stable_order(M, tokens, per_token, experts, kind):
    rng = np.random.default_rng(tokens + experts)
    ids = X.ids_of(rng, tokens, per_token, experts, kind)
    o = M.expert_sort(X.dev(ids), experts)
    want = X.order(ids, experts)
    for name, got, ref in zip(("offsets", "pair_of_row", "row_of_pair"), (o.offsets, o.pair_of_row, o.row_of_pair), want):
        assert np.array_equal(got.cpu().numpy(), ref), name


@pytest.mark.parametrize("kind", ["spread", "hot", "dropped", "none"])
@pytest.mark.parametrize("tokens,per_token,experts", [(9001, 8, 4096), (150001, 7, 3), (131073, 8, 130)])
def test_sort_of_many_pairs(M, tokens, per_token, experts, kind):
    test_sort_is_the_stable_order(M, tokens, per_token, experts, kind)


def test_sort_of_no_tokens(M):
    import torch

    o = M.expert_sort(torch.empty(0, 4, dtype=torch.int32, device="cuda"), 9)
    assert o.offsets.tolist() == [0] * 10 and o.pair_of_row.numel() == 0
    x = torch.empty(0, 16, device="cuda")
    assert M.expert_dispatch(x, o).shape == (0, 16) and M.expert_combine(x, o).shape == (0, 16)
    d_rows, d_w = M.expert_combine_backward(x, x, o)
    assert d_rows.shape == (0, 16) and d_w.shape == (0, 4)


def test_sort_extreme_ids(M):
    ids = np.array([[-2 ** 31, 2 ** 31 - 1, 0], [3, 4, -1]], np.int32)
    o = M.expert_sort(X.dev(ids), 4)
    assert o.offsets.tolist() == [0, 1, 1, 1, 2]
    assert o.pair_of_row.tolist() == [2, 3, -1, -1, -1, -1]
    assert o.row_of_pair.tolist() == [[-1, -1, 0], [1, -1, -1]]


SHAPES = [(1, 1, 1, 8), (1, 8, 128, 7168), (5, 3, 4, 1), (17, 2, 9, 33), (40, 8, 60, 513), (9, 11, 5, 520), (130, 6, 64, 2048),
          (12, 9, 16, 4104), (3, 17, 8, 2051)]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,per_token,experts,dim", SHAPES)
def test_there_and_back(M, tokens, per_token, experts, dim, kind, f32):
    import torch

    rng = np.random.default_rng(dim + tokens)
    ids = X.ids_of(rng, tokens, per_token, experts, kind)
    offsets, pair, row = X.order(ids, experts)
    n, pairs = int(offsets[-1]), tokens * per_token
    o = M.expert_sort(X.dev(ids), experts)
    x, x64 = rows_of(rng, tokens, dim, f32)
    left = torch.full((pairs, dim), -3.0, dtype=x.dtype, device="cuda")
    xs = M.expert_dispatch(x, o, out=left)
    assert xs is left
    assert np.array_equal(X.host(xs[:n]), x64[pair[:n] // per_token])
    assert (xs[n:] == -3).all()

    ys, y64 = rows_of(rng, pairs, dim, f32)
    ys[n:] = float("nan")  # never read
    w = rng.random((tokens, per_token)).astype(np.float32)
    wk = np.where(row < 0, np.nan, w).astype(np.float32)  # nor a weight without a row
    for weights, w64 in ((X.dev(wk), w.astype(np.float64)), (None, np.ones_like(w, np.float64))):
        got = X.host(M.expert_combine(ys, o, weights))
        has = (row >= 0)[..., None]
        terms = np.where(has, w64[..., None] * y64[np.maximum(row, 0)], 0)
        want, size = terms.sum(1), np.abs(terms).sum(1)
        tol = per_token * X.F32_ROUND * size * 1.01 + type_round(f32) * np.abs(want) * 1.01
        assert (np.abs(got - want) <= tol + 1e-45).all(), np.abs(got - want).max()

        g, g64 = rows_of(rng, tokens, dim, f32)
        d_left = torch.full((pairs, dim), -3.0, dtype=x.dtype, device="cuda")
        d_rows, d_w = M.expert_combine_backward(g, ys, o, weights, out=d_left)
        want = w64.reshape(-1)[pair[:n], None] * g64[pair[:n] // per_token]
        assert (np.abs(X.host(d_rows[:n]) - want) <= (X.F32_ROUND + type_round(f32)) * np.abs(want) * 1.01).all()
        assert (d_rows[n:] == -3).all()
        terms = np.where(has, g64[:, None] * y64[np.maximum(row, 0)], 0)
        depth = 8 * (-(-dim // 2048)) + 18
        assert (np.abs(X.host(d_w) - terms.sum(-1)) <= depth * X.F32_ROUND * np.abs(terms).sum(-1) * 1.01).all()

    ds, d64 = rows_of(rng, pairs, dim, f32)
    d_x = X.host(M.expert_dispatch_backward(ds, o))
    terms = np.where((row >= 0)[..., None], d64[np.maximum(row, 0)], 0)
    tol = per_token * X.F32_ROUND * np.abs(terms).sum(1) + type_round(f32) * np.abs(terms.sum(1))
    assert (np.abs(d_x - terms.sum(1)) <= tol * 1.01).all()


def test_gradients_are_those_of_differences(M):
    # combine is linear in the rows and in the weights, so a difference
    # quotient of its dot product with g is exact up to the f32 sums
    import torch

    rng = np.random.default_rng(11)
    tokens, per_token, experts, dim = 7, 3, 4, 40
    ids = X.ids_of(rng, tokens, per_token, experts, "dropped")
    o = M.expert_sort(X.dev(ids), experts)
    n = int(o.offsets[-1])
    ys, _ = rows_of(rng, tokens * per_token, dim, True)
    g, g64 = rows_of(rng, tokens, dim, True)
    w = torch.rand(tokens, per_token, device="cuda")
    d_rows, d_w = M.expert_combine_backward(g, ys, o, w)
    loss = lambda y, w: float((X.host(M.expert_combine(y, o, w)) * g64).sum())
    size = float(np.abs(X.host(M.expert_combine(ys.abs(), o, w)) * np.abs(g64)).sum())
    tol = 4 * (per_token + 1) * X.F32_ROUND * (size + np.abs(g64).sum())  # two sums, each off by at most this over 2
    for t in range(tokens):
        for j in range(per_token):
            up, down = w.clone(), w.clone()
            up[t, j] += 0.5
            down[t, j] -= 0.5
            step = float(up[t, j].double() - down[t, j].double())
            assert abs((loss(ys, up) - loss(ys, down)) / step - float(d_w[t, j])) <= 2 * tol
    for r in (0, n // 2, n - 1):
        for c in (0, 17, dim - 1):
            up, down = ys.clone(), ys.clone()
            up[r, c] += 0.5
            down[r, c] -= 0.5
            step = float(up[r, c].double() - down[r, c].double())
            assert abs((loss(up, w) - loss(down, w)) / step - float(d_rows[r, c])) <= 2 * tol
    # and of the dispatch: <dispatch(x), ds> = <x, dispatch_backward(ds)>
    x, x64 = rows_of(rng, tokens, dim, True)
    ds, d64 = rows_of(rng, tokens * per_token, dim, True)
    left = float((X.host(M.expert_dispatch(x, o)[:n]) * d64[:n]).sum())
    right = float((x64 * X.host(M.expert_dispatch_backward(ds, o))).sum())
    assert abs(left - right) <= per_token * X.F32_ROUND * np.abs(x64).sum() * np.abs(d64).max() * per_token


@pytest.mark.parametrize("f32", [False, True])
def test_row_strides_and_addresses(M, f32):
    import torch

    rng = np.random.default_rng(5)
    ids = X.ids_of(rng, 21, 4, 6, "hot")
    o = M.expert_sort(X.dev(ids), 6)
    offsets, pair, row = X.order(ids, 6)
    dt = torch.float32 if f32 else torch.bfloat16
    for dim, pad, start in ((64, 8, 8), (64, 3, 1), (30, 2, 2)):
        def wide(n):
            t, t64 = rows_of(rng, n, dim, f32)
            buf = torch.full((n, dim + pad + start), float("nan"), dtype=dt, device="cuda")
            buf[:, start:start + dim] = t
            return buf[:, start:start + dim], t64

        (x, x64), (ys, y64) = wide(21), wide(84)
        out = torch.zeros(84, dim + 5, dtype=dt, device="cuda")
        M.expert_dispatch(x, o, out=out[:, 2:2 + dim])
        assert np.array_equal(X.host(out[:, 2:2 + dim]), x64[pair // 4])
        assert (out[:, :2] == 0).all() and (out[:, 2 + dim:] == 0).all()
        got = X.host(M.expert_combine(ys, o))
        terms = y64[row]
        assert (np.abs(got - terms.sum(1)) <= (4 * X.F32_ROUND * np.abs(terms).sum(1) + type_round(f32) * np.abs(terms.sum(1))) * 1.01).all()
        d_rows, d_w = M.expert_combine_backward(x, ys, o, out=out[:, 2:2 + dim])
        assert np.array_equal(X.host(d_rows), x64[pair // 4])
        assert (out[:, :2] == 0).all() and (out[:, 2 + dim:] == 0).all()


def test_dispatch_keeps_every_bit(M):
    import torch

    bits = torch.arange(-2 ** 15, 2 ** 15, device="cuda").to(torch.int16).view(torch.bfloat16).reshape(32, 2048)
    o = M.expert_sort(torch.arange(32, dtype=torch.int32, device="cuda").flip(0).reshape(32, 1).contiguous(), 32)
    for x in (bits, bits[:, 1:]):
        assert torch.equal(M.expert_dispatch(x, o).view(torch.int16), x.flip(0).contiguous().view(torch.int16))


def test_two_calls_give_the_same_bits(M):
    import torch

    rng = np.random.default_rng(9)
    ids = X.dev(X.ids_of(rng, 3000, 6, 64, "hot"))
    w = torch.rand(3000, 6, device="cuda")
    ys, g = (torch.randn(n, 264, device="cuda", dtype=torch.bfloat16) for n in (18000, 3000))
    runs = []
    for _ in range(2):
        o = M.expert_sort(ids, 64)
        runs.append([o.offsets, o.pair_of_row, o.row_of_pair, M.expert_combine(ys, o, w),
                     *M.expert_combine_backward(g, ys, o, w)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_maps_out_of_range_have_no_row(M):
    import torch

    row = torch.tensor([[0, -5], [7, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    o = M.ExpertOrder(torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                      torch.tensor([0, -1, -1, -1], dtype=torch.int32, device="cuda"), row, experts=1)
    x = torch.ones(2, 16, device="cuda")
    xs = M.expert_dispatch(x, o, out=torch.zeros(4, 16, device="cuda"))
    assert (xs[0] == 1).all() and (xs[1:] == 0).all()
    assert (M.expert_combine(xs, o)[1] == 0).all()
    assert M.expert_combine_backward(x, xs, o)[1].tolist() == [[16.0, 0.0], [0.0, 0.0]]


def test_other_streams_and_graph_replays(M):
    import torch

    rng = np.random.default_rng(12)
    T, K, E, dim = 700, 8, 40, 264
    ids = X.dev(X.ids_of(rng, T, K, E, "dropped"))
    x, w = torch.randn(T, dim, device="cuda", dtype=torch.bfloat16), torch.rand(T, K, device="cuda")
    rows = torch.zeros(T * K, dim, device="cuda", dtype=torch.bfloat16)

    def step(stream=None):
        o = M.expert_sort(ids, E, stream=stream)
        xs = M.expert_dispatch(x, o, out=rows, stream=stream)
        out = M.expert_combine(xs, o, w, stream=stream)
        d_rows, d_w = M.expert_combine_backward(x, xs, o, w, stream=stream)
        return out, d_w, o.pair_of_row

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (s, s.cuda_stream):
        got = step(stream)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for i in range(3):
        ids.copy_(X.dev(X.ids_of(rng, T, K, E, KINDS[i])))
        x.copy_(torch.randn(T, dim, device="cuda"))
        rows.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        rows.zero_()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
