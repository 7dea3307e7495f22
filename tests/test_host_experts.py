"""Argument checks of the MXFP4 and routed-expert entry points on the host:
every refusal comes before a GPU call, with its status and a message."""
import ctypes as C

import pytest
from hypothesis import HealthCheck, given, settings
from hypothesis import strategies as st

import minirun_hip as M

AT = 1 << 32  # an address that no refused call reads
REFUSED = {M.INVALID_SHAPE, M.INVALID_ARGUMENT, M.INVALID_DTYPE, M.WORKSPACE_TOO_SMALL}


@pytest.fixture(scope="module")
def lib():
    return M.load()


def refused(status, want, *words):
    assert status == want, (status, M.last_error())
    assert all(w in M.last_error() for w in words), M.last_error()


def shape(*dims):
    return (C.c_int64 * len(dims))(*dims)


def validate(lib, packed, scales, pdt=M.U32, sdt=M.U8):
    ex, rows, cols = C.c_int64(-1), C.c_int64(-1), C.c_int64(-1)
    st = lib.mr_mxfp4_validate(pdt, len(packed), shape(*packed), sdt, len(scales), shape(*scales), C.byref(ex),
                               C.byref(rows), C.byref(cols))
    return st, (ex.value, rows.value, cols.value)


def test_validate(lib):
    assert validate(lib, (7, 8), (7, 2)) == (M.OK, (0, 7, 64))
    assert validate(lib, (3, 7, 8), (3, 7, 2)) == (M.OK, (3, 7, 64))
    assert validate(lib, (0, 4), (0, 1)) == (M.OK, (0, 0, 32))
    refused(validate(lib, (7, 8), (7, 2), pdt=M.F32)[0], M.INVALID_DTYPE, "uint32")
    refused(validate(lib, (7, 8), (7, 2), sdt=M.BF16)[0], M.INVALID_DTYPE, "uint8")
    refused(validate(lib, (8,), (2,))[0], M.INVALID_SHAPE, "rank")
    refused(validate(lib, (3, 7, 8), (7, 2))[0], M.INVALID_SHAPE, "rank")
    refused(validate(lib, (7, 8), (6, 2))[0], M.INVALID_SHAPE, "disagree")
    refused(validate(lib, (3, 7, 8), (2, 7, 2))[0], M.INVALID_SHAPE, "disagree")
    refused(validate(lib, (7, 8), (7, 1))[0], M.INVALID_SHAPE, "blocks of 32")
    refused(validate(lib, (7, 6), (7, 1))[0], M.INVALID_SHAPE, "blocks of 32")
    refused(validate(lib, (0, 7, 8), (0, 7, 2))[0], M.INVALID_SHAPE)
    refused(validate(lib, (7, 0), (7, 0))[0], M.INVALID_SHAPE)
    refused(lib.mr_mxfp4_validate(M.U32, 2, None, M.U8, 2, None, None, None, None), M.INVALID_ARGUMENT)


def test_quantize_refusals(lib):
    q = lambda x=AT, dt=M.BF16, rows=4, cols=64, ld=64, p=AT, s=AT: lib.mr_mxfp4_quantize(x, dt, rows, cols, ld, p, s, None)
    for cols in (0, -32, 33, 48):
        refused(q(cols=cols, ld=64), M.INVALID_SHAPE, "32")
    refused(q(rows=-1), M.INVALID_SHAPE)
    refused(q(rows=2 ** 40), M.INVALID_SHAPE, "2^37")
    for dt in (M.F16, M.U32, M.U8, 99, -1):
        refused(q(dt=dt), M.INVALID_DTYPE, "bf16 or f32")
    for kw in ({"x": None}, {"p": None}, {"s": None}):
        refused(q(**kw), M.INVALID_ARGUMENT, "non-NULL")
    refused(q(ld=63), M.INVALID_ARGUMENT, "stride")
    refused(q(x=AT + 1), M.INVALID_ARGUMENT, "misaligned")
    refused(q(x=AT + 2, dt=M.F32), M.INVALID_ARGUMENT, "misaligned")
    refused(q(p=AT + 2), M.INVALID_ARGUMENT, "misaligned")
    assert q(rows=0, x=None) == M.OK


def test_dequantize_refusals(lib):
    def d(packed=AT, scales=AT, rows=4, cols=64, out=AT, dt=M.BF16, ld=64):
        return lib.mr_mxfp4_dequantize(C.byref(M.MXFP4Desc(packed, scales, rows, cols)), out, dt, ld, None)

    refused(lib.mr_mxfp4_dequantize(None, AT, M.BF16, 64, None), M.INVALID_ARGUMENT)
    refused(d(cols=40), M.INVALID_SHAPE)
    refused(d(rows=-2), M.INVALID_SHAPE)
    refused(d(dt=M.F16), M.INVALID_DTYPE)
    for kw in ({"packed": None}, {"scales": None}, {"out": None}, {"ld": 32}, {"packed": AT + 2}, {"out": AT + 1}):
        refused(d(**kw), M.INVALID_ARGUMENT)
    assert d(rows=0, out=None) == M.OK


def w_desc(packed=AT, scales=AT, rows=64, cols=96):
    return C.byref(M.MXFP4Desc(packed, scales, rows, cols))


def test_matmul_refusals(lib):
    def mm(x=AT, dt=M.BF16, t=4, ld=96, y=AT, ydt=M.BF16, ldy=64, **w):
        return lib.mr_mxfp4_matmul(x, dt, t, ld, w_desc(**w), y, ydt, ldy, None)

    refused(lib.mr_mxfp4_matmul(AT, M.BF16, 4, 96, None, AT, M.BF16, 64, None), M.INVALID_ARGUMENT)
    for kw in ({"cols": 80}, {"cols": 0}, {"rows": 0}, {"rows": -4}, {"rows": 2 ** 22 + 1}, {"cols": 2 ** 20 + 32}, {"t": -1}):
        refused(mm(**kw), M.INVALID_SHAPE)
    for kw in ({"dt": M.F16}, {"dt": M.U8}, {"dt": 77}, {"ydt": M.F16}, {"ydt": M.U32}):
        refused(mm(**kw), M.INVALID_DTYPE)
    refused(mm(dt=M.U32), M.INVALID_DTYPE, "mr_mxfp4_matmul_quantized")
    for kw in ({"x": None}, {"y": None}, {"packed": None}, {"scales": None}):
        refused(mm(**kw), M.INVALID_ARGUMENT, "non-NULL")
    for kw in ({"x": AT + 8}, {"packed": AT + 4}, {"ld": 100}, {"ld": 98, "dt": M.F32}):
        refused(mm(**kw), M.INVALID_ARGUMENT, "16")
    for kw in ({"ld": 88}, {"ldy": 63}, {"y": AT + 1}, {"y": AT + 2, "ydt": M.F32}, {"ld": 2 ** 22 + 8}, {"ld": 2 ** 41}, {"ldy": 2 ** 41}):
        refused(mm(**kw), M.INVALID_ARGUMENT)
    assert mm(t=0, x=None, y=None) == M.OK


def test_quantized_matmul_refusals(lib):
    def mm(y=AT, ydt=M.BF16, ldy=64, x=w_desc(rows=4), **w):
        return lib.mr_mxfp4_matmul_quantized(x, w_desc(**w), y, ydt, ldy, None)

    refused(mm(x=None), M.INVALID_ARGUMENT)
    refused(mm(cols=64), M.INVALID_SHAPE, "columns")
    refused(mm(x=w_desc(rows=2 ** 31)), M.INVALID_SHAPE)
    refused(mm(ydt=M.F16), M.INVALID_DTYPE)
    for kw in ({"x": w_desc(packed=None)}, {"x": w_desc(scales=None)}, {"y": None}, {"x": w_desc(packed=AT + 4)}, {"ldy": 63}):
        refused(mm(**kw), M.INVALID_ARGUMENT)
    assert mm(x=w_desc(rows=0), y=None) == M.OK


def test_expert_matmul_refusals(lib):
    def mm(w=None, **kw):
        a = M.MXFP4ExpertArgs()
        a.x, a.x_dtype, a.x_stride, a.x_rows = AT, M.BF16, 96, 4
        a.w = M.MXFP4Desc(AT, AT, 64, 96)
        a.experts, a.offsets, a.pair_of_row, a.per_token, a.rows = 8, AT, AT, 2, 8
        a.y, a.y_dtype, a.y_stride = AT, M.BF16, 64
        for k, v in (w or {}).items():
            setattr(a.w, k, v)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.mr_mxfp4_expert_matmul(C.byref(a), None)

    refused(lib.mr_mxfp4_expert_matmul(None, None), M.INVALID_ARGUMENT)
    for kw in ({"experts": 0}, {"experts": 4097}, {"rows": -2}, {"rows": 2 ** 24 + 2}, {"rows": 7}, {"per_token": 0},
               {"x_rows": 8}, {"pair_of_row": None}, {"w": {"cols": 72}}, {"w": {"rows": 0}},
               {"rows": 2 ** 23, "x_rows": 2 ** 22, "w": {"cols": 512}, "x_stride": 512},
               {"w": {"rows": 2 ** 22}, "rows": 2 ** 24, "x_rows": 2 ** 23, "y_stride": 2 ** 22}):
        refused(mm(**kw), M.INVALID_SHAPE)
    for kw in ({"x_dtype": M.F16}, {"y_dtype": M.U32}):
        refused(mm(**kw), M.INVALID_DTYPE)
    for kw in ({"x": None}, {"y": None}, {"offsets": None}, {"offsets": AT + 2}, {"pair_of_row": AT + 1}, {"x": AT + 4},
               {"x_scales": AT}, {"x_dtype": M.U32}, {"x_stride": 90}, {"y_stride": 60}, {"w": {"packed": None}}):
        refused(mm(**kw), M.INVALID_ARGUMENT)
    assert mm(rows=0, x_rows=0, x=None, y=None) == M.OK


def test_sort_sizes_and_refusals(lib):
    size = lib.mr_expert_sort_workspace_size
    assert size(256, 8, 128) == 0  # one workgroup
    assert size(257, 8, 128) == 2 * 128 * 4
    assert size(1 << 21, 8, 4096) == 8192 * 4096 * 4
    assert size(0, 8, 16) == 0
    for bad in ((-1, 1, 1), (1, 0, 1), (1, -3, 1), (1, 1, 0), (1, 1, 4097), ((1 << 21) + 1, 8, 4), (2 ** 31 - 1, 2 ** 31 - 1, 4)):
        assert size(*bad) == 0
        refused(lib.mr_expert_sort(AT, *bad, AT, AT, AT, AT, 1 << 40, None), M.INVALID_SHAPE)
    sort = lambda ids=AT, o=AT, p=AT, r=AT, ws=AT, n=1 << 30, t=600: lib.mr_expert_sort(ids, t, 8, 16, o, p, r, ws, n, None)
    for kw in ({"ids": None}, {"o": None}, {"p": None}, {"r": None}):
        refused(sort(**kw), M.INVALID_ARGUMENT, "non-NULL")
    for kw in ({"ids": AT + 1}, {"o": AT + 2}, {"p": AT + 3}, {"r": AT + 2}, {"ws": AT + 2}):
        refused(sort(**kw), M.INVALID_ARGUMENT, "misaligned")
    refused(sort(n=127), M.WORKSPACE_TOO_SMALL, "required")
    refused(sort(ws=None), M.WORKSPACE_TOO_SMALL)


def test_row_refusals(lib):
    dispatch = lambda x=AT, dt=M.BF16, t=4, dim=64, ld=64, m=AT, k=2, out=AT, lo=64: lib.mr_expert_dispatch(
        x, dt, t, dim, ld, m, k, out, lo, None)
    combine = lambda x=AT, dt=M.BF16, t=4, dim=64, ld=64, m=AT, k=2, out=AT, lo=64, w=None: lib.mr_expert_combine(
        x, dt, ld, dim, m, w, t, k, out, lo, None)
    backward = lambda x=AT, dt=M.BF16, t=4, dim=64, ld=64, m=AT, k=2, out=AT, lo=64, w=None, y=AT, dw=AT: \
        lib.mr_expert_combine_backward(x, dt, ld, dim, y, 64, m, w, t, k, out, lo, dw, None)
    for call in (dispatch, combine, backward):
        refused(call(t=-1), M.INVALID_SHAPE)
        refused(call(k=0), M.INVALID_SHAPE)
        refused(call(t=2 ** 23, k=3), M.INVALID_SHAPE, "2^24")
        refused(call(dim=0, ld=0, lo=0), M.INVALID_SHAPE)
        refused(call(dim=2 ** 24 + 1, ld=2 ** 25, lo=2 ** 25), M.INVALID_SHAPE)
        refused(call(t=2 ** 23, k=1, dim=2 ** 20, ld=2 ** 20, lo=2 ** 20), M.INVALID_SHAPE, "one launch")
        for dt in (M.F16, M.I32, 99):
            refused(call(dt=dt), M.INVALID_DTYPE)
        for kw in ({"x": None}, {"m": None}, {"ld": 63}, {"lo": 63}, {"ld": 2 ** 41}, {"x": AT + 1}, {"out": AT + 1}, {"m": AT + 2}):
            refused(call(**kw), M.INVALID_ARGUMENT)
        assert call(t=0, x=None) == M.OK
    for call in (dispatch, combine):
        refused(call(out=None), M.INVALID_ARGUMENT)
    for call in (combine, backward):
        refused(call(w=AT + 2), M.INVALID_ARGUMENT)
    refused(backward(y=None), M.INVALID_ARGUMENT)
    refused(backward(dw=AT + 1), M.INVALID_ARGUMENT)
    assert backward(out=None, dw=None, x=None) == M.OK  # nothing asked for


def test_python_checks_come_before_the_library():
    import torch

    cpu = torch.zeros(4, 64)
    for call in (lambda: M.mxfp4_quantize(cpu), lambda: M.expert_sort(torch.zeros(4, 2, dtype=torch.int32), 3),
                 lambda: M.ExpertOrder(*(torch.zeros(4, dtype=torch.int32),) * 3, experts=3),
                 lambda: M.MXFP4Weights(torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.uint8))):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    with pytest.raises(M.MRError, match="uint8"):
        M.MXFP4Weights(torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32))


def test_rows_of_a_tensor_need_a_stride():
    """Repeated rows (stride 0) have no row stride that the library takes: it is
    passed on as it is, and refused; one row may have any."""
    import torch

    class OnGPU(torch.Tensor):
        is_cuda = True

    def stride(t):
        return M._rows2d(t.as_subclass(OnGPU), "x")

    assert stride(torch.zeros(1, 64).expand(3, 64)) == 0
    assert stride(torch.zeros(1, 64)) == 64
    assert stride(torch.zeros(5, 64)[::5]) == 320
    assert stride(torch.zeros(64).as_strided((1, 64), (0, 1))) == 64
    assert stride(torch.zeros(3, 80)[:, :64]) == 80
    with pytest.raises(ValueError):
        stride(torch.zeros(3, 1).expand(3, 64))


# ---------------------------------------------------------------- random arguments
dim = st.one_of(st.integers(-5, 4200), st.sampled_from([0, 1, 32, 64, 4096, 2 ** 24, 2 ** 31 - 1, -2 ** 31]))
wide = st.one_of(st.integers(-5, 70000), st.sampled_from([0, 32, 2 ** 20, 2 ** 22, 2 ** 37, 2 ** 62, -2 ** 63, 2 ** 63 - 1]))
dtype = st.integers(-1, 7)
RANDOM = settings(max_examples=300, deadline=None, derandomize=True, suppress_health_check=[HealthCheck.too_slow])


def nothing_or_refused(status, nothing):
    """With NULL buffers: refused with a message, or there was nothing to do."""
    assert status == M.OK and nothing or status in REFUSED and M.last_error(), status


@RANDOM
@given(rows=wide, cols=wide, dt=dtype, ld=wide, experts=dim, tokens=dim)
def test_mxfp4_checks_of_random_arguments(lib, rows, cols, dt, ld, experts, tokens):
    w = M.MXFP4Desc(None, None, rows, cols)
    x = M.MXFP4Desc(None, None, tokens, cols)
    nothing_or_refused(lib.mr_mxfp4_quantize(None, dt, rows, cols, ld, None, None, None), rows == 0)
    nothing_or_refused(lib.mr_mxfp4_dequantize(C.byref(w), None, dt, ld, None), rows == 0)
    nothing_or_refused(lib.mr_mxfp4_matmul(None, dt, tokens, ld, C.byref(w), None, M.F32, ld, None), tokens == 0)
    nothing_or_refused(lib.mr_mxfp4_matmul_quantized(C.byref(x), C.byref(w), None, dt, ld, None), tokens == 0)
    a = M.MXFP4ExpertArgs()
    a.x_dtype, a.x_stride, a.x_rows, a.w, a.experts, a.per_token, a.rows = dt, ld, tokens, w, experts, 1, tokens
    a.y_dtype, a.y_stride = M.BF16, ld
    nothing_or_refused(lib.mr_mxfp4_expert_matmul(C.byref(a), None), tokens == 0)
    ps, ss = shape(rows, cols), shape(rows, experts)
    status = lib.mr_mxfp4_validate(M.U32, 2, ps, M.U8, 2, ss, None, None, None)
    nothing_or_refused(status, 0 <= rows and 8 * cols == 32 * experts)


@RANDOM
@given(tokens=dim, per_token=dim, experts=dim, width=wide, dt=dtype, ld=wide)
def test_routing_checks_of_random_arguments(lib, tokens, per_token, experts, width, dt, ld):
    size = lib.mr_expert_sort_workspace_size(tokens, per_token, experts)
    assert 0 <= size <= 2 ** 24 // 2048 * 4096 * 4
    refused(lib.mr_expert_sort(None, tokens, per_token, experts, None, None, None, None, 0, None),
            M.INVALID_SHAPE if size == 0 and not (tokens >= 0 and per_token > 0 and tokens * per_token <= 2 ** 24
                                                  and 0 < experts <= 4096) else M.INVALID_ARGUMENT)
    none = tokens == 0
    nothing_or_refused(lib.mr_expert_dispatch(None, dt, tokens, width, ld, None, per_token, None, ld, None), none)
    nothing_or_refused(lib.mr_expert_combine(None, dt, ld, width, None, None, tokens, per_token, None, ld, None), none)
    nothing_or_refused(lib.mr_expert_combine_backward(None, dt, ld, width, None, ld, None, None, tokens, per_token, AT, ld,
                                                      None, None), none)
