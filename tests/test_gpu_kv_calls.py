"""Calls of the paged cache from Python that its documentation allows or refuses: strides of
axes of one entry, numbers past 32 bits, a cache whose tensors would be exchanged."""
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


def test_numbers_past_32_bits_are_refused(M):
    """ctypes keeps the low 32 bits of a number, which would be another window or column."""
    import torch

    cache = M.KVCache.zeros(2, 1, 16, 64)
    q = torch.zeros(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    table, lens = ints(0).reshape(1, 1), ints(5)
    trig = torch.zeros(1, 4, device="cuda")
    k = torch.zeros(1, 1, 64, device="cuda")
    bad = [lambda n: M.kv_attention(q, cache, table, lens, scale=1.0, window=n),
           lambda n: M.kv_attention(q, cache, table, lens, scale=1.0, max_kv_len=n),
           lambda n: M.head_norm_rope(q, cos_t=trig, sin_t=trig, col0=n),
           lambda n: M.head_norm_rope_backward(q, q, cos_t=trig, sin_t=trig, col0=n),
           lambda n: M.kv_append(cache, k, k, ints(0), cos_t=trig, sin_t=trig, col0=n)]
    for i, call in enumerate(bad):
        for n in (2 ** 32, 2 ** 32 + 3, 2 ** 31, -2 ** 32, 2 ** 70):
            with pytest.raises((M.MRError, TypeError, ValueError)):
                call(n)
                print("accepted", i, n)


def test_sizes_past_32_bits_are_refused(M):
    """2^32 + 1 tokens or heads (of one row in memory) are not one."""
    import torch

    many = 2 ** 32 + 1
    one = torch.ones(1, 1, 8, device="cuda", dtype=torch.bfloat16)
    out = torch.zeros(1, 1, 8, device="cuda", dtype=torch.bfloat16)
    with pytest.raises((M.MRError, ValueError)):
        M.head_norm_rope(one.expand(many, 1, 8), q_out=out.expand(many, 1, 8))
    with pytest.raises((M.MRError, ValueError)):
        M.head_norm_rope(one, one.expand(1, many, 8), k_out=out.expand(1, many, 8))
    assert (out == 0).all()


@pytest.mark.parametrize("mxfp4", [False, True])
def test_a_cache_keeps_its_tensors(M, mxfp4):
    """What calls take lies behind the addresses that the cache was made with."""
    import torch

    cache = M.KVCache.zeros(2, 1, 16, 64, mxfp4=mxfp4)
    for name in ("k", "v", "k_scales", "v_scales", "pages", "page_size", "kv_heads", "head_dim", "device"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(4, 1, 16, 64, device="cuda"))
    cache.k += 1  # (in place: the same tensor)
    assert (cache.k == 1).all()
    assert cache.k.shape[0] == cache.pages == 2 and cache.head_dim == 64 and (cache.k_scales is not None) == mxfp4
