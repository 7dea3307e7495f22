"""Host-side checks of the head-norm, cache-append and paged-attention entry points at the
edges of what they take (test_host_kv.py has the refusals)."""
import ctypes as C

import pytest

import minirun_hip as M
from test_host_kv import AT, FAR, append_args, attention_args, norm_args, refused


@pytest.fixture(scope="module")
def lib():
    return M.load()


def test_strides_of_axes_of_one_entry_are_not_read(lib):
    """The calls get as far as their workspaces, or their missing slots."""
    odd = [7, -1, FAR + 1]
    for s in odd:
        heads = dict(q_head_stride=s, out_head_stride=s, cache=dict(kv_heads=1, page_stride=32 * 64), heads=1)
        long = dict(max_pages=4096)
        refused(lib.mr_kv_attention(C.byref(attention_args(**heads, **long)), None), M.WORKSPACE_TOO_SMALL)
        tokens = dict(q_token_stride=s, out_token_stride=s, tokens=1, batch=1)
        refused(lib.mr_kv_attention(C.byref(attention_args(**tokens, **long)), None), M.WORKSPACE_TOO_SMALL)
        one = dict(tokens=1, q__x_token_stride=s, q__out_token_stride=s, q__d_out_token_stride=s, k__x_token_stride=s,
                   k__out_token_stride=s, k__d_out_token_stride=s)
        refused(lib.mr_head_norm_rope_backward(C.byref(norm_args(**one)), None), M.WORKSPACE_TOO_SMALL)
        one = dict(q__heads=1, k__heads=1, q__x_head_stride=s, q__out_head_stride=s, q__d_out_head_stride=s, k__x_head_stride=s,
                   k__out_head_stride=s, k__d_out_head_stride=s)
        refused(lib.mr_head_norm_rope_backward(C.byref(norm_args(**one)), None), M.WORKSPACE_TOO_SMALL)
        for one in (dict(tokens=1, k_token_stride=s, v_token_stride=s),
                    dict(cache=dict(kv_heads=1, pages=0, k=None, v=None), k_head_stride=s, v_head_stride=s)):
            args = append_args(**{"cache": dict(pages=0, k=None, v=None), **one})
            assert lib.mr_kv_append(C.byref(args), None) == M.OK


def test_more_workgroups_than_a_launch_takes(lib):
    """A launch has fewer than 2^32 threads: 2^24 workgroups of few queries, 2^23 of prompts.  (Without
    `out` nothing is launched: what passes the sizes is refused for that.)"""
    call = lambda **kw: lib.mr_kv_attention(C.byref(attention_args(**kw, out=None, q_offsets=AT)), None)
    heads = dict(heads=8, cache=dict(kv_heads=8, page_stride=8 * 32 * 64))
    # 65 rows of a sequence and key head: a tile for each, one more for the average
    for batch, ok in ((10 ** 6, False), (830000, True)):
        refused(call(batch=batch, tokens=65 * batch, **heads), *((M.INVALID_ARGUMENT, "non-NULL") if ok else (M.INVALID_SHAPE, "launch")))
    wide = dict(heads=8, cache=dict(kv_heads=8, head_dim=160, page_stride=8 * 32 * 160))
    refused(call(batch=10 ** 6, tokens=65 * 10 ** 6, **wide), M.INVALID_ARGUMENT, "non-NULL")
    for batch, ok in ((2 ** 21, False), (10 ** 6, True)):
        refused(call(batch=batch, tokens=batch, **heads), *((M.INVALID_ARGUMENT, "non-NULL") if ok else (M.INVALID_SHAPE, "launch")))
    # parts do not count: a call that they would take past a launch has fewer of them
    long = dict(heads=32, cache=dict(kv_heads=32, page_stride=32 * 32 * 64), max_pages=2 ** 15)
    refused(lib.mr_kv_attention(C.byref(attention_args(batch=1024, tokens=1024, **long, out=None)), None), M.INVALID_ARGUMENT, "non-NULL")


def test_every_workgroup_of_the_gradients_has_rows(lib):
    """A workgroup, whose sums take a row of the workspace, has 4 waves of 64 / lanes groups that take 2 rows a step."""
    for dim, lanes in ((128, 16), (64, 8), (33, 8), (512, 64), (8, 1)):
        step = 4 * (64 // lanes) * 2
        for tokens, q, k in ((1, 1, 0), (1, 32, 4), (300, 6, 2), (777, 12, 2), (5000, 3, 1), (100000, 32, 8)):
            a = M.HeadNormArgs(tokens, dim, M.HeadRows(q), M.HeadRows(k))
            rows = lib.mr_head_norm_rope_backward_workspace_size(C.byref(a)) // (4 * dim)
            assert 0 < rows <= min(-(-tokens * q // step) + -(-tokens * k // step), 1026), (dim, tokens, q, k, rows)
