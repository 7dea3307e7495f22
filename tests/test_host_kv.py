"""Argument checks of the head-norm, cache-append and paged-attention entry points on
the host: every refusal comes before a GPU call, with its status and a message; and
what their workspaces cover."""
import ctypes as C

import pytest
from hypothesis import HealthCheck, given, settings
from hypothesis import strategies as st

import minirun_hip as M

AT = 1 << 32  # an address that no refused call reads
REFUSED = {M.INVALID_SHAPE, M.INVALID_ARGUMENT, M.INVALID_DTYPE, M.WORKSPACE_TOO_SMALL}
FAR = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return M.load()


def put(a, **fields):
    for name, value in fields.items():
        at, *parts = a, *name.split("__")
        for p in parts[:-1]:
            at = getattr(at, p)
        setattr(at, parts[-1], value)
    return a


def refused(status, want, *words):
    assert status == want, (status, M.last_error())
    assert all(w in M.last_error() for w in words), M.last_error()


def norm_args(**fields):
    a = M.HeadNormArgs()
    put(a, tokens=5, dim=64, x_dtype=M.BF16, weight_dtype=M.F32, out_dtype=M.BF16, eps=1e-6)
    for rows, heads in ((a.q, 4), (a.k, 2)):
        put(rows, heads=heads, x=AT, out=AT, weight=AT, d_out=AT, d_weight=AT + 256 * heads, x_token_stride=64 * heads, x_head_stride=64,
            out_token_stride=64 * heads, out_head_stride=64, d_out_token_stride=64 * heads, d_out_head_stride=64)
    put(a.rope, cos_t=AT, sin_t=AT, positions=AT, table_rows=9, dim=32)
    return put(a, **fields)


def test_head_norm_refusals(lib):
    for f in (lib.mr_head_norm_rope, lib.mr_head_norm_rope_backward):
        call = lambda **kw: f(C.byref(norm_args(**kw)), None)
        refused(f(None, None), M.INVALID_ARGUMENT, "NULL")
        for kw in (dict(tokens=-1), dict(dim=0), dict(dim=513), dict(q__heads=-1), dict(q__heads=0, k__heads=0),
                   dict(tokens=2 ** 31 - 1), dict(tokens=2 ** 25, q__heads=40, dim=8), dict(tokens=2 ** 24, dim=512, q__heads=4)):
            refused(call(**kw), M.INVALID_SHAPE)
        for kw in (dict(x_dtype=M.F16), dict(out_dtype=M.U8), dict(weight_dtype=77), dict(x_dtype=-1)):
            refused(call(**kw), M.INVALID_DTYPE, "bf16 or f32")
        for eps in (-1.0, float("nan"), float("inf")):
            refused(call(eps=eps), M.INVALID_ARGUMENT, "eps")
        for kw in (dict(rope__dim=33), dict(rope__dim=-2), dict(rope__dim=66), dict(rope__col0=33), dict(rope__col0=-1),
                   dict(rope__col0=2 ** 31 - 1), dict(rope__table_rows=0), dict(rope__positions=None, rope__table_rows=4)):
            refused(call(**kw), M.INVALID_SHAPE, "rota")
        for kw in (dict(rope__pairs=2), dict(rope__cos_t=None), dict(rope__sin_t=None), dict(rope__sin_t=AT + 2),
                   dict(rope__positions=AT + 1), dict(q__x=None), dict(k__out=None), dict(q__x=AT + 1),
                   dict(k__weight=AT + 2), dict(q__x_head_stride=-1), dict(q__x_token_stride=FAR + 1), dict(q__out_head_stride=63),
                   dict(k__out_token_stride=127), dict(q__out_head_stride=0), dict(q__out_token_stride=0, q__out_head_stride=64)):
            refused(call(**kw), M.INVALID_ARGUMENT)
    call = lambda **kw: lib.mr_head_norm_rope_backward(C.byref(norm_args(**kw)), None)
    refused(call(q__d_out=None), M.INVALID_ARGUMENT, "NULL")
    refused(call(q__d_weight=AT, k__d_weight=AT), M.INVALID_ARGUMENT, "one d_weight")
    refused(call(q__d_out_token_stride=-1), M.INVALID_ARGUMENT, "stride")
    refused(call(), M.WORKSPACE_TOO_SMALL, "workspace")
    refused(call(workspace_bytes=1 << 20), M.INVALID_ARGUMENT, "workspace")
    refused(call(workspace_bytes=1 << 20, workspace=AT + 2), M.INVALID_ARGUMENT, "workspace")


def test_head_norm_without_work(lib):
    assert lib.mr_head_norm_rope(C.byref(norm_args(tokens=0, q__x=None)), None) == M.OK
    a = norm_args(tokens=0, q__d_weight=None, k__d_weight=None)
    assert lib.mr_head_norm_rope_backward(C.byref(a), None) == M.OK
    size = lib.mr_head_norm_rope_backward_workspace_size
    assert size(None) == 0 and size(C.byref(norm_args(dim=0))) == 0 and size(C.byref(norm_args(tokens=0))) == 0
    one, many = size(C.byref(norm_args(tokens=1))), size(C.byref(norm_args(tokens=1 << 20)))
    assert one == 2 * 64 * 4 and 512 * 64 * 4 <= many <= 1026 * 64 * 4


def cache_of(a, mxfp4=False, **fields):
    put(a, k=AT, v=AT, pages=8, page_size=32, kv_heads=2, head_dim=64, page_stride=32 * 2 * 64 // (8 if mxfp4 else 1))
    if mxfp4:
        put(a, k_scales=AT, v_scales=AT, scale_page_stride=32 * 2 * 2)
    return put(a, **fields)


BAD_CACHES = [
    (M.INVALID_SHAPE, dict(pages=-1)), (M.INVALID_SHAPE, dict(page_size=0)), (M.INVALID_SHAPE, dict(page_size=24)),
    (M.INVALID_SHAPE, dict(page_size=-16)), (M.INVALID_SHAPE, dict(kv_heads=0)), (M.INVALID_SHAPE, dict(head_dim=48)),
    (M.INVALID_SHAPE, dict(head_dim=288)), (M.INVALID_SHAPE, dict(head_dim=0)), (M.INVALID_SHAPE, dict(page_size=2 ** 30)),
    (M.INVALID_SHAPE, dict(pages=2 ** 27)), (M.INVALID_SHAPE, dict(kv_heads=2 ** 20)),
    (M.INVALID_ARGUMENT, dict(page_stride=100)), (M.INVALID_ARGUMENT, dict(page_stride=-4096)),
    (M.INVALID_ARGUMENT, dict(page_stride=FAR * 2)), (M.INVALID_ARGUMENT, dict(page_stride=4096 + 2)),
    (M.INVALID_ARGUMENT, dict(k=None)), (M.INVALID_ARGUMENT, dict(v=None)), (M.INVALID_ARGUMENT, dict(k=AT + 8)),
]
BAD_MX = [(M.INVALID_ARGUMENT, dict(k_scales=None)), (M.INVALID_ARGUMENT, dict(v_scales=None)),
          (M.INVALID_ARGUMENT, dict(scale_page_stride=127)), (M.INVALID_ARGUMENT, dict(scale_page_stride=FAR + 1))]


def append_args(mxfp4=False, cache={}, **fields):
    a = M.KVAppendArgs()
    cache_of(a.cache, mxfp4, **cache)
    put(a, tokens=5, k=AT, v=AT, dtype=M.BF16, slots=AT, normalize=1, norm_w=AT, norm_w_dtype=M.F32, eps=1e-6,
        k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
    put(a.rope, cos_t=AT, sin_t=AT, positions=AT, table_rows=9, dim=32)
    return put(a, **fields)


def test_append_refusals(lib):
    f = lib.mr_kv_append
    call = lambda *a, **kw: f(C.byref(append_args(*a, **kw)), None)
    refused(f(None, None), M.INVALID_ARGUMENT, "NULL")
    for want, kw in BAD_CACHES:
        refused(call(cache=kw), want)
    for want, kw in BAD_MX:
        refused(call(True, cache=kw), want)
    for kw in (dict(tokens=-1), dict(tokens=2 ** 28), dict(rope__dim=31), dict(rope__col0=33), dict(rope__table_rows=-1)):
        refused(call(**kw), M.INVALID_SHAPE)
    for kw in (dict(dtype=M.F16), dict(norm_w_dtype=M.U8)):
        refused(call(**kw), M.INVALID_DTYPE)
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(slots=AT + 2), dict(k=AT + 1), dict(norm_w=AT + 1),
               dict(eps=-1.0), dict(k_head_stride=-64), dict(v_token_stride=FAR + 1), dict(rope__pairs=-1)):
        refused(call(**kw), M.INVALID_ARGUMENT)
    assert call(tokens=0, k=None) == M.OK and call(cache=dict(pages=0, k=None, v=None)) == M.OK


def attention_args(mxfp4=False, cache={}, **fields):
    a = M.KVAttentionArgs()
    cache_of(a.cache, mxfp4, **cache)
    put(a, batch=3, tokens=3, heads=8, q=AT, q_token_stride=512, q_head_stride=64, page_table=AT, page_table_stride=8, max_pages=8,
        kv_lens=AT, scale=0.1, out=AT, out_dtype=M.BF16, out_token_stride=512, out_head_stride=64)
    return put(a, **fields)


def test_attention_refusals(lib):
    f, size = lib.mr_kv_attention, lib.mr_kv_attention_workspace_size
    call = lambda *a, **kw: f(C.byref(attention_args(*a, **kw)), None)
    refused(f(None, None), M.INVALID_ARGUMENT, "NULL")
    assert size(None) == 0
    for want, kw in BAD_CACHES:
        refused(call(cache=kw), want)
        assert size(C.byref(attention_args(cache=kw))) == 0
    for want, kw in BAD_MX:
        refused(call(True, cache=kw), want)
    for kw in (dict(batch=-1), dict(tokens=-1), dict(heads=0), dict(heads=7), dict(heads=-8), dict(tokens=4), dict(max_pages=-1),
               dict(max_pages=2 ** 27), dict(max_kv_len=-1), dict(window=-1), dict(tokens=2 ** 30, q_offsets=AT),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
               dict(scale=3e38),
               dict(batch=2 ** 24, tokens=2 ** 24)):
        refused(call(**kw), M.INVALID_SHAPE)
    refused(call(out_dtype=M.F16), M.INVALID_DTYPE)
    for kw in (dict(q=None), dict(out=None), dict(kv_lens=None), dict(page_table=None), dict(q=AT + 8), dict(out=AT + 8),
               dict(q_head_stride=68), dict(q_token_stride=-512), dict(out_head_stride=32), dict(out_token_stride=0),
               dict(out_token_stride=516), dict(page_table=AT + 2), dict(kv_lens=AT + 1), dict(q_offsets=AT + 2),
               dict(sinks=AT + 2), dict(lse=AT + 1), dict(page_table_stride=-1), dict(page_table_stride=FAR + 1)):
        refused(call(**kw), M.INVALID_ARGUMENT)
    assert call(batch=0, tokens=0, q=None) == M.OK and call(tokens=0, q_offsets=AT, q=None) == M.OK
    long = dict(max_pages=4096)
    need = size(C.byref(attention_args(**long)))
    assert need > 0 and size(C.byref(attention_args())) == 0
    refused(call(**long), M.WORKSPACE_TOO_SMALL, str(need))
    refused(call(**long, workspace=AT, workspace_bytes=need - 1), M.WORKSPACE_TOO_SMALL)
    refused(call(**long, workspace_bytes=need), M.INVALID_ARGUMENT, "workspace")
    refused(call(**long, workspace=AT + 4, workspace_bytes=need), M.INVALID_ARGUMENT, "workspace")
    # counted in 32 bits, past the keys by a few tiles
    most = dict(max_pages=2 ** 25, page_table_stride=2 ** 25, max_kv_len=100)
    refused(call(**{**most, "max_pages": 2 ** 25 + 1}), M.INVALID_SHAPE, "pages")
    refused(call(**most, out=None), M.INVALID_ARGUMENT)
    refused(call(tokens=2 ** 27 + 1, q_offsets=AT), M.INVALID_SHAPE, "tokens")
    refused(call(tokens=2 ** 27, q_offsets=AT, out=None), M.INVALID_ARGUMENT)
    # a hint or a window below the least part of a split: no workspace
    assert size(C.byref(attention_args(**long, max_kv_len=300))) == 0
    assert size(C.byref(attention_args(**long, window=300))) == 0


I32 = st.one_of(st.integers(-2 ** 31, 2 ** 31 - 1), st.integers(-2, 70), st.sampled_from([0, 16, 32, 64, 128, 256]))
I64 = st.one_of(st.integers(-2 ** 63, 2 ** 63 - 1), st.integers(-1, 600))


def fill(draw, a):
    for name, kind in a._fields_:
        if isinstance(getattr(a, name), C.Structure):
            fill(draw, getattr(a, name))
        elif kind is C.c_float:
            setattr(a, name, draw(st.sampled_from([0.0, 1.0, -1.0, float("nan"), 1e-6])))
        elif kind in (C.c_int32, C.c_int):
            setattr(a, name, draw(I32))
        elif kind is C.c_int64:
            setattr(a, name, draw(I64))
        elif kind is C.c_size_t:
            setattr(a, name, draw(st.sampled_from([0, 64, 2 ** 40])))
        # pointers stay NULL: nothing can run


@settings(max_examples=300, deadline=None, suppress_health_check=list(HealthCheck))
@given(st.data())
def test_random_arguments_are_refused_or_have_no_work(lib, data):
    for kind, f, sizes in ((M.HeadNormArgs, lib.mr_head_norm_rope, None), (M.KVAppendArgs, lib.mr_kv_append, None),
                           (M.HeadNormArgs, lib.mr_head_norm_rope_backward, lib.mr_head_norm_rope_backward_workspace_size),
                           (M.KVAttentionArgs, lib.mr_kv_attention, lib.mr_kv_attention_workspace_size)):
        a = kind()
        fill(data.draw, a)
        if sizes:
            sizes(C.byref(a))
        status = f(C.byref(a), None)
        if status == M.OK:
            assert a.tokens == 0 or a.batch == 0 if kind is M.KVAttentionArgs else a.tokens == 0 or a.cache.pages == 0
        else:
            assert status in REFUSED, (status, M.last_error())
