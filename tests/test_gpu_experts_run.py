"""MXFP4 and routing calls in use: a training step of a layer of experts run
eagerly, captured, on two streams at once and from several host threads; what
lies behind the outputs; buffers past 32-bit byte offsets."""
import threading

import numpy as np
import pytest

import mxfp4_inputs as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


class Step:
    """Tokens to their experts, both projections, back, and the gradients of the
    routing, over inputs of its own; every output whole."""

    def __init__(self, M, seed, tokens=700, per_token=8, experts=60, hidden=512, inner=416, f32=False):
        import torch

        self.M, self.E, self.n = M, experts, tokens * per_token
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
        dt = torch.float32 if f32 else torch.bfloat16
        self.ids = torch.empty(tokens, per_token, dtype=torch.int32, device="cuda")
        self.x, self.d_out = rand(tokens, hidden).to(dt), rand(tokens, hidden).to(dt)
        self.router = torch.rand(tokens, per_token, device="cuda", generator=g)
        self.up = M.mxfp4_quantize(rand(experts, inner, hidden))
        self.down = M.mxfp4_quantize(rand(experts, hidden, inner))
        self.h = torch.zeros(self.n, inner, device="cuda", dtype=torch.bfloat16)
        self.y = torch.zeros(self.n, hidden, device="cuda", dtype=dt)
        self.d_rows = torch.zeros(self.n, hidden, device="cuda", dtype=dt)
        self.fill(seed)

    def fill(self, seed):
        import torch

        g = torch.Generator(device="cuda").manual_seed(1000 + seed)
        shape = self.ids.shape
        self.ids.copy_(torch.randint(-3, self.E + 3, shape, device="cuda", generator=g, dtype=torch.int32))
        self.x.copy_(torch.randn(self.x.shape, device="cuda", generator=g))

    def run(self, stream=None):
        M = self.M
        o = M.expert_sort(self.ids, self.E, stream=stream)
        xs = M.mxfp4_quantize(self.x, stream=stream)
        h = M.mxfp4_expert_mm(xs, self.up, o, out=self.h, stream=stream)
        y = M.mxfp4_expert_mm(h, self.down, o, sorted_rows=True, out=self.y, stream=stream)
        out = M.expert_combine(y, o, self.router, stream=stream)
        d_rows, d_weights = M.expert_combine_backward(self.d_out, y, o, self.router, out=self.d_rows, stream=stream)
        d_x = M.expert_dispatch_backward(d_rows, o, stream=stream)
        return [o.offsets, o.pair_of_row, o.row_of_pair, h, y, out, d_rows, d_weights, d_x]

    def reset(self):
        for t in (self.h, self.y, self.d_rows):
            t.zero_()

    def eager(self):
        self.reset()
        return [t.clone() for t in self.run()]


def same(got, want):
    import torch

    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("f32", [False, True])
def test_two_captured_steps_replayed_together(M, f32):
    import torch

    steps = [Step(M, 1, f32=f32), Step(M, 2, tokens=300, experts=1030, f32=f32)]  # (the second's counts are scanned)
    for s in steps:
        s.eager()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for turn in range(4):
        for i, s in enumerate(steps):
            s.fill(10 * turn + i)
        want = [s.eager() for s in steps]
        for s in steps:
            s.reset()
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        assert all(same(o, w) for o, w in zip(outs, want)), turn


def test_threads_on_their_own_streams(M):
    import torch

    steps = [Step(M, 20 + i, tokens=200 + 150 * i) for i in range(4)]
    want = [s.eager() for s in steps]
    for s in steps:
        s.reset()
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            for _ in range(5):
                r = steps[i].run(stream)
            with torch.cuda.stream(stream):
                got[i] = [t.clone() for t in r]
            stream.synchronize()
        except Exception as e:  # noqa: BLE001  (reported by the test's thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and all(same(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,cols,pad", [(1, 32, 0), (33, 512, 0), (3, 2080, 8), (1, 7168, 0), (5, 4096, 64), (257, 96, 0)])
def test_nothing_behind_the_outputs_is_written(M, rows, cols, pad, f32):
    import torch

    lib, dt = M.load(), torch.float32 if f32 else torch.bfloat16
    x = torch.randn(rows, cols + pad, device="cuda").to(dt)[:, :cols]
    n, guard = rows * cols, 70000
    packed = torch.full((n // 8 + guard,), 0x5A5A5A5A, dtype=torch.int32, device="cuda")
    scales = torch.full((n // 32 + guard,), 77, dtype=torch.uint8, device="cuda")
    M._check(lib.mr_mxfp4_quantize(x.data_ptr(), M._dtype_code(dt), rows, cols, cols + pad, packed.data_ptr(),
                                   scales.data_ptr(), M._stream(None)))
    w = M.mxfp4_quantize(x.contiguous())
    assert torch.equal(packed[:n // 8], w.packed.view(-1)) and torch.equal(scales[:n // 32], w.scales.view(-1))
    assert (packed[n // 8:] == 0x5A5A5A5A).all() and (scales[n // 32:] == 77).all()
    ld = cols + pad
    out = torch.full((rows * ld + guard,), -5.0, dtype=dt, device="cuda")
    M._check(lib.mr_mxfp4_dequantize(M.C.byref(w.desc()), out.data_ptr(), M._dtype_code(dt), ld, M._stream(None)))
    body = out[:rows * ld].view(rows, ld)
    assert torch.equal(body[:, :cols], M.mxfp4_dequantize(w, dt))
    assert (body[:, cols:] == -5).all() and (out[rows * ld:] == -5).all()


def test_rows_past_32_bit_offsets(M):
    # 300,000 rows of 16 KB: 4.9 GB, each token's value in all of its row
    import torch

    tokens, per_token, experts, dim = 150000, 2, 5, 8192
    ids = X.ids_of(np.random.default_rng(1), tokens, per_token, experts, "spread")
    o = M.expert_sort(X.dev(ids), experts)
    x = (torch.arange(tokens, device="cuda") % 251).to(torch.bfloat16)[:, None].expand(tokens, dim).contiguous()
    rows = M.expert_dispatch(x, o)
    pair = o.pair_of_row.long()
    n = int(o.offsets[-1])
    want = (pair[:n] // per_token % 251).to(torch.bfloat16)
    for c in (0, 1, 4097, dim - 1):
        assert torch.equal(rows[:n, c], want)
    out = M.expert_combine(rows, o)
    count = (o.row_of_pair >= 0).sum(1)
    for c in (0, 5000, dim - 1):
        assert torch.equal(out[:, c], (x[:, c].float() * count).to(torch.bfloat16))
    d_rows, d_w = M.expert_combine_backward(x, rows, o)
    assert torch.equal(d_rows[:n, dim - 1], want) and torch.equal(d_rows[:n, 3], want)
    exact = torch.where(o.row_of_pair >= 0, (x[:, :1].double() ** 2 * dim).expand(tokens, per_token), 0.0)
    # a sum of 8192 equal whole numbers below 2^16: up to 64 roundings of 2^-24 each
    assert (d_w.double() - exact).abs().max() <= 64 * 2 ** -24 * 250 ** 2 * dim


@pytest.mark.parametrize("kind", ["bf16", "mxfp4"])
def test_products_past_32_bit_offsets(M, kind):
    # y of 40,000 x 32,776 in f32: 5.2 GB
    import torch

    tokens, out, inp = 40000, 32776, 32
    w = M.mxfp4_quantize(torch.ones(out, inp, device="cuda") * 2 ** (torch.arange(out, device="cuda") % 7)[:, None])
    scale = 2.0 ** (torch.arange(tokens, device="cuda") % 5)
    x = scale[:, None].expand(tokens, inp).to(torch.bfloat16).contiguous()
    y = M.mxfp4_mm(M.mxfp4_quantize(x) if kind == "mxfp4" else x, w, out_dtype=torch.float32)
    for t in (0, 1, 32767, 32768, 39998, 39999):
        assert torch.equal(y[t], 32 * scale[t] * 2.0 ** (torch.arange(out, device="cuda") % 7)), t


def test_quantized_values_past_32_bits(M):
    import torch

    rows, cols = 131080, 32768  # 2^32 + 2^18 values
    x = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    at = [(0, 0), (65535, 32767), (131071, 5), (131072, 0), (131079, 32767)]
    for r, c in at:
        x[r, c] = 1.5
    w = M.mxfp4_quantize(x)
    assert int((w.packed != 0).sum()) == len(at) and int((w.scales != 0).sum()) == len(at)
    back = M.mxfp4_dequantize(w, torch.bfloat16)
    assert int((back != 0).sum()) == len(at) and all(float(back[r, c]) == 1.5 for r, c in at)
