"""Calls of the paged cache from Python that its documentation allows: strides of axes of one entry."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def ints(*v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("tokens,heads", [(1, 4), (3, 1), (1, 1)])
def test_strides_of_axes_of_one_entry(M, tokens, heads):
    """Nothing is a stride away along an axis of one entry, whatever the stride says."""
    import torch

    rng = np.random.default_rng(2)
    dim = 64
    pages = K.Pages(rng, 4, 1, 16, dim, True)
    cache = pages.device(M)
    q, _ = K.values_of(rng, (tokens, heads, dim), False)
    odd = (heads * dim if tokens > 1 else 12345, dim if heads > 1 else 77, 1)
    strange = torch.as_strided(q, q.shape, odd)
    table, lens = ints(0, 1).reshape(1, 2).expand(tokens, 2), torch.full((tokens,), 25, dtype=torch.int32, device="cuda")
    want = M.kv_attention(q, cache, table, lens, scale=0.1)
    out = torch.zeros_like(want)
    assert torch.equal(M.kv_attention(strange, cache, table, lens, scale=0.1), want)
    M.kv_attention(strange, cache, table, lens, scale=0.1, out=torch.as_strided(out, out.shape, odd))
    assert torch.equal(out, want)
    norm = M.head_norm_rope(q)
    assert torch.equal(M.head_norm_rope(strange), norm)
    M.head_norm_rope(strange, q_out=torch.as_strided(out, out.shape, odd))
    assert torch.equal(out, norm)
    if heads == 1:
        a, b = M.KVCache.zeros(1, 1, 16, dim), M.KVCache.zeros(1, 1, 16, dim)
        slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
        M.kv_append(a, q, q, slots)
        M.kv_append(b, strange, strange, slots)
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
