"""Host-side checks of the head-norm, cache-append and paged-attention entry points at the
edges of what they take (test_host_kv.py has the refusals)."""
import ctypes as C

import pytest

import minirun_hip as M
from test_host_kv import FAR, append_args, attention_args, norm_args, refused


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
