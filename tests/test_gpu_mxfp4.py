"""MXFP4 quantisation on the GPU, bit for bit against the plain rule: every
rounding tie, the ends of the scale range, subnormal values, signed zeros, NaN
and infinities, odd numbers of rows and blocks, row strides and addresses that
the wide loads do not take."""
import numpy as np
import pytest

import mxfp4_inputs as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def quantized(M, x, f32):
    import torch

    t = X.dev(x if f32 else X.to_bf16(x))
    w = M.mxfp4_quantize(t)
    torch.cuda.synchronize()
    return w


def check(M, x, f32, tag):
    seen = np.asarray(x, np.float32) if f32 else X.from_bf16(X.to_bf16(x))
    packed, scales = X.quantize(seen)
    w = quantized(M, x, f32)
    assert np.array_equal(w.scales.cpu().numpy(), scales), f"{tag}: scale bytes"
    assert np.array_equal(w.packed.cpu().numpy().view(np.uint32), packed), f"{tag}: words"


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 7168), (3, 64), (5, 96), (7, 2080), (33, 512), (2, 16384), (301, 1536)])
def test_random_rows(M, rows, cols, f32):
    rng = np.random.default_rng(rows * cols)
    x = (rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-30, 30, (rows, 1)))).astype(np.float32)
    x[rng.random(x.shape) < 0.01] *= 100
    check(M, x, f32, f"{rows}x{cols}")


@pytest.mark.parametrize("f32", [False, True])
def test_every_tie_at_every_scale(M, f32):
    # a block whose largest value is 4 2^e .. 7.5 2^e, and the numbers between
    # two e2m1 neighbours, their ends and the middle, which is a tie
    steps = np.array([0, 0.125, 0.25, 0.375, 0.5, 0.75, 0.875, 1.25, 1.125, 1.75, 2.5, 2.25, 3.5, 3.25, 5, 4.5])
    x = []
    for e in range(-127, 126):
        block = np.concatenate([steps, -steps])
        block[0] = (4, 5, 6, 7, 7.5)[e % 5]
        x.append(block * 2.0 ** e)
    x = np.array(x)
    keep = np.abs(x).max(1) < 3e38
    check(M, x[keep].astype(np.float32), f32, "ties")


@pytest.mark.parametrize("f32", [False, True])
def test_zeros_subnormals_and_blocks_that_are_not_finite(M, f32):
    tiny = 2.0 ** -149 if f32 else 2.0 ** -133
    rng = np.random.default_rng(3)
    x = rng.standard_normal((9, 96)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2, :32] = tiny * np.arange(32)
    x[3] *= np.float32(2.0 ** -126)
    x[4, 40] = np.nan
    x[5, 64] = np.inf
    x[6, 0], x[6, 95] = -np.inf, np.nan
    x[7, :64] = 3.3e38
    w = quantized(M, x, f32)
    check(M, x, f32, "special")
    v = X.host(M.mxfp4_dequantize(w))
    seen = np.asarray(x, np.float32) if f32 else X.from_bf16(X.to_bf16(x))
    bad = ~np.isfinite(seen.reshape(9, 3, 32)).all(-1)
    assert np.array_equal(np.isnan(v.reshape(9, 3, 32)).all(-1), bad)  # whole blocks, and no others
    assert np.array_equal(np.isnan(v.reshape(9, 3, 32)).any(-1), bad)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("pad,start", [(8, 0), (8, 8), (3, 0), (5, 1), (4, 4)])
def test_row_strides_and_addresses(M, pad, start, f32):
    import torch

    rng = np.random.default_rng(pad)
    x = rng.standard_normal((13, 160)).astype(np.float32)
    buf = torch.full((13, 160 + pad + start), float("nan"), dtype=torch.float32 if f32 else torch.bfloat16, device="cuda")
    buf[:, start:start + 160] = X.dev(x if f32 else X.to_bf16(x))
    w = M.mxfp4_quantize(buf[:, start:start + 160])
    packed, scales = X.quantize(x if f32 else X.from_bf16(X.to_bf16(x)))
    assert np.array_equal(w.packed.cpu().numpy().view(np.uint32), packed)
    assert np.array_equal(w.scales.cpu().numpy(), scales)


def test_vector_and_stack(M):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((3, 5, 64)).astype(np.float32)
    w = M.mxfp4_quantize(X.dev(x))
    assert (w.experts, w.rows, w.cols) == (3, 5, 64)
    packed, scales = X.quantize(x.reshape(15, 64))
    assert np.array_equal(w.packed.cpu().numpy().view(np.uint32).reshape(15, 8), packed)
    v = M.mxfp4_dequantize(w)
    assert tuple(v.shape) == (3, 5, 64)
    assert np.array_equal(X.host(v).reshape(15, 64), X.values(packed, scales))
    one = M.mxfp4_quantize(X.dev(x[1, 2]))
    assert (one.rows, one.cols) == (1, 64) and np.array_equal(one.packed.cpu().numpy().view(np.uint32)[0], packed[7])
    empty = M.mxfp4_quantize(X.dev(x[0, :0]))
    assert empty.rows == 0 and M.mxfp4_dequantize(empty).shape == (0, 64)


@pytest.mark.parametrize("f32", [False, True])
def test_dequantize_every_byte_and_code(M, f32):
    import torch

    # row b: byte b, each code twice
    packed = np.tile(np.array([0x76543210, 0xFEDCBA98] * 2, np.uint32), (256, 1))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    got = X.host(M.mxfp4_dequantize(w, dtype=torch.float32 if f32 else torch.bfloat16))
    want = X.values(packed, scales)
    big = np.abs(want) > (3.4028234663852886e38 if f32 else 3.3895313892515355e38)
    want = np.where(big, np.copysign(np.inf, want), want)
    assert np.array_equal(got, want, equal_nan=True)


def test_dequantize_into_rows_of_a_wider_matrix(M):
    import ctypes as C
    import torch

    rng = np.random.default_rng(6)
    packed, scales = X.matrix(rng, 11, 96)
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    for start, width in ((0, 128), (8, 104), (1, 99)):
        for dt in (torch.bfloat16, torch.float32):
            out = torch.full((11, width), -7.0, dtype=dt, device="cuda")
            view = out[:, start:start + 96]
            M._check(M.load().mr_mxfp4_dequantize(C.byref(w.desc()), M._ptr(view), M._dtype_code(dt), width, M._stream(None)))
            assert np.array_equal(X.host(view), X.values(packed, scales))
            out[:, start:start + 96] = -7
            assert (out == -7).all()


def test_quantized_values_are_within_half_a_step(M):
    # e2m1 steps are 2^-2 of the value at most between 0.5 2 and 4, and the
    # scaled value is below 8: a value v of a block with power p is off by at
    # most max(|v| / 4, p / 4), or by up to 2 p where it is above 6 p
    rng = np.random.default_rng(8)
    x = rng.standard_normal((64, 512)).astype(np.float32)
    w = M.mxfp4_quantize(X.dev(x))
    v, p = X.host(M.mxfp4_dequantize(w)), np.repeat(X.power(w.scales.cpu().numpy()), 32, 1)
    limit = np.where(np.abs(x) > 6 * p, 2 * p, np.maximum(np.abs(x) / 4, p / 4))
    assert (np.abs(v - x) <= limit).all()


def test_graph_replays_follow_new_inputs(M):
    import torch

    x = torch.randn(5, 256, device="cuda", dtype=torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        M.mxfp4_dequantize(M.mxfp4_quantize(x))
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w = M.mxfp4_quantize(x)
        v = M.mxfp4_dequantize(w)
    for i in range(3):
        x.copy_(torch.randn(5, 256, device="cuda") * 3 ** i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(v, M.mxfp4_dequantize(M.mxfp4_quantize(x)))
