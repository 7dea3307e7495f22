"""The gradients of head norms where a workgroup walks over many rows: values at sizes of
several steps, with whole and partial last ones, heads that divide a step and heads that do not;
in place; and the gradient of a weight whose side has no heads.

The oracle is test_gpu_head_norm.py's formula in f64 on the GPU, with its tolerances."""
import ctypes as C

import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def turned(x, cos, sin, col0, halves, inverse=False):
    """kv_inputs.turn for f64 tensors; cos, sin [tokens, n]."""
    y, n = x.clone(), cos.shape[1]
    if not n:
        return y
    a = slice(col0, col0 + n) if halves else slice(col0, col0 + 2 * n, 2)
    b = slice(col0 + n, col0 + 2 * n) if halves else slice(col0 + 1, col0 + 2 * n, 2)
    c, s = cos[:, None].double(), sin[:, None].double() * (-1 if inverse else 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def check(dx, dw, dy, x, w, cos, sin, col0, halves, f32):
    """kv_inputs.norm_backward's values and bounds.  A weight's chain of sums at these sizes: 14
    roundings of a term, at most 16 rows of a lane, 6 + 4 of a workgroup, 16 + 64 partial rows (so
    a row that is left out or taken twice, a 10^5th of a sum here, is seen)."""
    import torch

    x, dy, w = x.double(), dy.double(), w.double()
    g = turned(dy, cos, sin, col0, halves, inverse=True)
    # |a cos| + |b sin|, whichever of the two signs a turn has
    around = torch.maximum(turned(dy.abs(), cos.abs(), sin.abs(), col0, halves), turned(dy.abs(), cos.abs(), -sin.abs(), col0, halves))
    r = ((x * x).mean(-1, keepdim=True) + EPS).rsqrt()
    unit = x * r
    gw = g * w
    dot = (gw * unit).mean(-1, keepdim=True)
    want = r * (gw - unit * dot)
    bound = r * (15 * around * w.abs() + 54 * unit.abs() * (around * (w * unit).abs()).mean(-1, keepdim=True))
    off = (dx.double() - want).abs() - K.U * bound - (X.F32_ROUND if f32 else X.BF16_ROUND) * want.abs() - 1e-37
    assert (off <= 0).all(), off.argmax()
    want_w, total = (g * unit).sum((0, 1)), (around * unit.abs()).sum((0, 1))
    off = (dw.double() - want_w).abs() - 120 * K.U * total - K.U * want_w.abs()
    assert (off <= 0).all(), off.argmax()


# tokens, heads, kv_heads, dim, rotated columns, first of them, halves
WALKS = [
    (4099, 8, 2, 128, 128, 0, True),   # a wave takes 8 rows a step: the heads of one token
    (3001, 7, 3, 512, 64, 448, False),  # a row is a wave; 7 and 3 heads wrap
    (30001, 5, 2, 64, 40, 12, True),   # rotations not in whole lanes
    (2500, 32, 8, 128, 128, 0, False),
    (30011, 3, 1, 33, 14, 3, False),   # values one by one
]


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("shape", WALKS)
def test_gradients_of_many_rows(M, shape, f32):
    import torch

    T, H, G, D, rope, col0, halves = shape
    # a workgroup leaves a row of sums, and takes 4 x (64 / lanes) x 2 rows a step
    sizes = M.HeadNormArgs(T, D, M.HeadRows(H), M.HeadRows(G))
    groups = M.load().mr_head_norm_rope_backward_workspace_size(C.byref(sizes)) // (4 * D)
    lanes = next(n for n in (1, 2, 4, 8, 16, 32, 64) if 8 * n >= D)
    assert T * (H + G) > groups * 512 // lanes
    gen = torch.Generator(device="cuda").manual_seed(T)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.float32 if f32 else torch.bfloat16)
    q, k, dq, dk, wq, wk = make(T, H, D) * 2, make(T, G, D) * 0.1, make(T, H, D), make(T, G, D), make(D), make(D)
    angle = torch.rand(T + 7, rope // 2, generator=gen, device="cuda") * 8 - 4
    positions = torch.randint(0, T + 7, (T,), generator=gen, device="cuda")
    cos, sin = angle.cos(), angle.sin()
    got = M.head_norm_rope_backward(dq, q, dk, k, q_weight=wq, k_weight=wk, eps=EPS, cos_t=cos, sin_t=sin,
                                    positions=positions.int(), col0=col0, halves=halves)
    at = cos[positions], sin[positions]
    check(got[0], got[2], dq, q, wq, *at, col0, halves, f32)
    check(got[1], got[3], dk, k, wk, *at, col0, halves, f32)


def args_of(M, q, dq, out, weight, d_weight, heads_k=0, k_weight=None, d_k_weight=None):
    T, H, D = q.shape
    rows = lambda t: (t.data_ptr(), *t.stride()[:2])
    a = M.HeadNormArgs(T, D, M.HeadRows(H, *rows(q), weight.data_ptr(), *rows(out), *rows(dq), d_weight.data_ptr()),
                       M.HeadRows(heads_k), M.BF16 if q.element_size() == 2 else M.F32, M.F32,
                       M.BF16 if out.element_size() == 2 else M.F32, EPS)
    if k_weight is not None:
        a.k.weight, a.k.d_weight = k_weight.data_ptr(), d_k_weight.data_ptr()
    return a


def call(M, a):
    import torch

    lib = M.load()
    n = lib.mr_head_norm_rope_backward_workspace_size(C.byref(a))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    M._check(lib.mr_head_norm_rope_backward(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("where", ["x", "d_out"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,H,D", [(3, 5, 96), (9001, 6, 128), (2001, 7, 33)])
def test_gradients_in_place(M, where, f32, T, H, D):
    """`out` is x itself, or d_out itself."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(D)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.float32 if f32 else torch.bfloat16)
    q, dq, w = make(T, H, D), make(T, H, D), torch.rand(D, generator=gen, device="cuda") + 0.5
    want, want_w = M.head_norm_rope_backward(dq, q, q_weight=w, eps=EPS)
    dw = torch.full((D,), float("nan"), device="cuda")
    out = q if where == "x" else dq
    call(M, args_of(M, q, dq, out, w, dw))
    assert torch.equal(out, want) and torch.equal(dw, want_w)


def test_a_side_without_heads_has_gradients_of_zero(M):
    """A weight whose side has no heads: its gradient is written like one of no tokens."""
    import torch

    T, H, D = 9, 4, 40
    q, dq, w = torch.randn(T, H, D, device="cuda"), torch.randn(T, H, D, device="cuda"), torch.ones(D, device="cuda")
    want, want_w = M.head_norm_rope_backward(dq, q, q_weight=w, eps=EPS)
    dw, dwk = (torch.full((D,), float("nan"), device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    call(M, args_of(M, q, dq, out, w, dw, 0, w, dwk))
    assert torch.equal(out, want) and torch.equal(dw, want_w) and (dwk == 0).all()
    # and from Python
    none = q[:, :0]
    torch.full((D,), float("nan"), device="cuda")  # (what the next vector of D may be found to hold)
    dx, dk, dw, dwk = M.head_norm_rope_backward(dq, q, none, none, q_weight=w, k_weight=w, eps=EPS)
    assert torch.equal(dx, want) and dk.shape == (T, 0, D) and torch.equal(dw, want_w) and (dwk == 0).all()
    dx, dk, dw, dwk = M.head_norm_rope_backward(none, none, dq, q, q_weight=w, k_weight=w, eps=EPS)
    assert torch.equal(dk, want) and torch.equal(dwk, want_w) and (dw == 0).all()


@pytest.mark.parametrize("dim", [96, 33])
def test_rows_whose_squares_pass_f32(M, dim):
    """Zeros, as the header says, and gradients of zeros; the other rows are as without them."""
    import torch

    x, dy = torch.randn(5, 2, dim, device="cuda"), torch.randn(5, 2, dim, device="cuda")
    want, (dx, _) = M.head_norm_rope(x, eps=EPS), M.head_norm_rope_backward(dy, x, eps=EPS)
    x[2, 1] *= 1e20
    got, (gx, _) = M.head_norm_rope(x, eps=EPS), M.head_norm_rope_backward(dy, x, eps=EPS)
    want[2, 1], dx[2, 1] = 0, 0
    assert torch.equal(got, want) and torch.equal(gx, dx)
