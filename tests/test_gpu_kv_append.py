"""Keys and values into the pages of a cache on the GPU.  Stored values are rounded
once from the exact ones, so they are compared bit for bit with what 64 bits give (two
64-bit computations differ by 2^-50 or so, and of the 10^6 values here none lies that
near a border)."""
import numpy as np
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


def stored(cache):
    """The cache's tensors as host arrays."""
    parts = [cache.k, cache.v] + ([cache.k_scales, cache.v_scales] if cache.k_scales is not None else [])
    out = []
    for t in parts:
        t = t.cpu().contiguous()
        out.append(t.view(__import__("torch").int16).numpy().view(np.uint16) if t.dtype.is_floating_point
                   else t.numpy().view(np.uint32) if t.dtype.itemsize == 4 else t.numpy())
    return out


def expect(pages, k, v, slots):
    """Host arrays of the pages with rows k, v (64 bits) put in."""
    parts = [pages.k.copy(), pages.v.copy()] + ([pages.ks.copy(), pages.vs.copy()] if pages.mxfp4 else [])
    n, heads, ps, dim = pages.shape
    for i, x in enumerate((k, v)):
        flat = x.reshape(-1, dim)
        rows = K.quantize64(flat) if pages.mxfp4 else (K.round_bf16(flat),)
        for part, r in zip(parts[i::2], rows):
            r = r.reshape(x.shape[0], heads, -1)
            for t, s in enumerate(slots):
                if 0 <= s < n * ps:
                    part[s // ps, :, s % ps] = r[t]
    return parts


# tokens, heads, dim, page size, normalised, rotated columns, first, halves
SHAPES = [
    (1, 1, 32, 16, True, 32, 0, True), (1, 4, 128, 16, True, 128, 0, True), (32, 4, 128, 16, True, 128, 0, False),
    (77, 2, 96, 48, True, 64, 32, False), (77, 2, 96, 48, True, 24, 8, True), (50, 3, 64, 32, False, 0, 0, False),
    (129, 1, 256, 64, False, 256, 0, True), (40, 2, 192, 16, True, 0, 0, False), (40, 2, 160, 80, True, 22, 3, True),
    (65, 5, 224, 32, False, 10, 5, False), (300, 8, 128, 128, True, 64, 64, True),
]


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_stored_rows(M, shape, f32, mxfp4):
    T, H, D, ps, normalize, rope, col0, halves = shape
    rng = np.random.default_rng([T, H, D, f32, mxfp4])
    n = -(-T // ps) + 2
    pages = K.Pages(rng, n, H, ps, D, mxfp4)
    k, k64 = K.values_of(rng, (T, H, D), f32, 3.0)
    v, v64 = K.values_of(rng, (T, H, D), f32, 0.3)
    slots = rng.permutation(n * ps)[:T].astype(np.int32)
    slots[rng.random(T) < 0.1] = rng.choice([-1, n * ps, 2 ** 31 - 1, -2 ** 31])
    w, w64 = K.values_of(rng, (D,), not f32)
    cos, sin = K.tables(rng, T + 9, rope // 2)
    positions = rng.integers(0, T + 9, T).astype(np.int32)
    how = dict(col0=col0, halves=halves)
    if normalize:
        weighted = T != 40
        how.update(normalize=True, eps=EPS, **({"norm_weight": w} if weighted else {}))
        k64 = K.norm(k64, w64 if weighted else 1.0, float(np.float32(EPS)))
    if rope:
        how.update(cos_t=X.dev(cos), sin_t=X.dev(sin), positions=X.dev(positions))
        k64 = K.turn(k64, cos[positions], sin[positions], col0, halves)
    cache = pages.device(M, gap=16 if T % 2 else 0)
    M.kv_append(cache, k, v, X.dev(slots), **how)
    names = ("k", "v", "k_scales", "v_scales")
    for name, got, want in zip(names, stored(cache), expect(pages, k64, v64, slots)):
        assert np.array_equal(got, want), (name, np.argwhere(got != want)[:3])
    if mxfp4:
        k_all, v_all = cache.values()
        kv = X.values(*stored(cache)[0::2]), X.values(*stored(cache)[1::2])
        assert np.array_equal(X.host(k_all), kv[0]) and np.array_equal(X.host(v_all), kv[1])


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-18, 1e-3, 1e3, 1e18, 1e30, 1e37])
def test_rows_of_any_size(M, scale, mxfp4):
    """Squares that leave f32's range, values near its ends, rows of zeros, and a large value in each third row:
    what the stored values are does not depend on how they were found."""
    rng = np.random.default_rng(5)
    T, H, D = 48, 2, 128
    x = (scale * rng.standard_normal((T, H, D))).astype(np.float32)
    x[::3, :, 7] *= 1e3 if scale < 1e34 else 1.0
    x[5] = 0
    w = rng.uniform(0.5, 1.5, D).astype(np.float32)
    cos, sin = K.tables(rng, T, D // 2)
    for normalize in (True, False):
        pages = K.Pages(rng, 4, H, 16, D, mxfp4)
        cache = pages.device(M)
        slots = rng.permutation(64)[:T].astype(np.int32)
        k64 = K.norm(x.astype(np.float64), w.astype(np.float64), float(np.float32(EPS))) if normalize else x.astype(np.float64)
        M.kv_append(cache, X.dev(x), X.dev(x), X.dev(slots), normalize=normalize, norm_weight=X.dev(w) if normalize else None,
                    eps=EPS, cos_t=X.dev(cos), sin_t=X.dev(sin), halves=True)
        for got, want in zip(stored(cache), expect(pages, K.turn(k64, cos, sin, 0, True), x.astype(np.float64), slots)):
            assert np.array_equal(got, want), np.argwhere(got != want)[:3]


@pytest.mark.parametrize("mxfp4", [False, True])
def test_values_next_to_a_border(M, mxfp4):
    """Values that lie on a border of the 4-bit (or bf16) grid, or next to one by less than f32 resolves."""
    D, T = 64, 40
    rng = np.random.default_rng(3)
    x = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8], (T, 1, D)).astype(np.float32)
    x[:, :, 0] = 4.0  # the block's power
    x[:, :, 32] = 4.0
    cos = np.full((T, D // 2), 1.0, np.float32)
    sin = (rng.choice([-1, 0, 1], (T, D // 2)) * 2.0 ** -40).astype(np.float32)  # moves a value by 2^-40 of its partner
    pages = K.Pages(rng, 3, 1, 16, D, mxfp4)
    cache = pages.device(M)
    slots = np.arange(T, dtype=np.int32)
    M.kv_append(cache, X.dev(x), X.dev(x), X.dev(slots), cos_t=X.dev(cos), sin_t=X.dev(sin), halves=True)
    k64 = K.turn(x.astype(np.float64), cos, sin, 0, True)
    for got, want in zip(stored(cache), expect(pages, k64, x.astype(np.float64), slots)):
        assert np.array_equal(got, want)


def test_infinities_and_nan(M):
    import torch

    D = 64
    for mxfp4 in (False, True):
        cache = M.KVCache.zeros(1, 1, 16, D, mxfp4=mxfp4)
        x = torch.ones(4, 1, D, device="cuda")
        x[1, 0, 3], x[2, 0, 40], x[3, 0, 0] = float("nan"), float("inf"), -3.4e38
        M.kv_append(cache, x, x, torch.arange(4, dtype=torch.int32, device="cuda"))
        k, v = cache.values()
        assert torch.equal(k.nan_to_num(nan=5.0, posinf=9.0), v.nan_to_num(nan=5.0, posinf=9.0))
        if mxfp4:  # a block is NaN whole, its neighbour is not
            assert torch.isnan(v[0, 0, 1, :32]).all() and torch.isfinite(v[0, 0, 1, 32:]).all()
            assert torch.isnan(v[0, 0, 2, 32:]).all() and torch.isfinite(v[0, 0, 2, :32]).all()
        else:
            assert torch.isnan(v[0, 0, 1, 3]) and torch.isinf(v[0, 0, 2, 40]) and torch.isfinite(v[0, 0, 1, 4:]).all()
        assert (v[0, 0, 0] == 1).all() and (v[0, 0, 4:] == 0).all()


def test_strided_rows_and_no_tokens(M):
    import torch

    rng = np.random.default_rng(9)
    T, H, D = 21, 2, 64
    fused, _ = K.values_of(rng, (T, 1 + 4 * H * D), False)  # rows off a 16-byte boundary
    k, v = fused[:, 1:1 + H * D].view(T, H, D), fused[:, 1 + 2 * H * D:1 + 3 * H * D].view(T, H, D)
    slots = torch.arange(T, dtype=torch.int32, device="cuda") + 3
    for mxfp4 in (False, True):
        a, b = (M.KVCache.zeros(2, H, 16, D, mxfp4=mxfp4) for _ in range(2))
        M.kv_append(a, k, v, slots, normalize=True)
        M.kv_append(b, k.contiguous(), v.contiguous(), slots, normalize=True)
        assert all(np.array_equal(x, y) for x, y in zip(stored(a), stored(b)))
        before = stored(a)
        M.kv_append(a, k[:0], v[:0], slots[:0])
        M.kv_append(a, k, v, torch.full_like(slots, -1))
        assert all(np.array_equal(x, y) for x, y in zip(stored(a), before))


def test_refusals(M):
    import torch

    cache = M.KVCache.zeros(2, 2, 16, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 8, device="cuda")
    bad = [
        lambda: M.kv_append(cache, k[:, :1], k, slots), lambda: M.kv_append(cache, k, k.bfloat16(), slots),
        lambda: M.kv_append(cache, k.half(), k.half(), slots), lambda: M.kv_append(cache, k, k, slots[:2]),
        lambda: M.kv_append(cache, k, k, slots.long()), lambda: M.kv_append(cache, k, k, slots.cpu()),
        lambda: M.kv_append(cache, k, k, slots, norm_weight=torch.ones(64, device="cuda")),
        lambda: M.kv_append(cache, k, k, slots, normalize=True, norm_weight=torch.ones(32, device="cuda")),
        lambda: M.kv_append(cache, k, k, slots, normalize=True, eps=float("inf")),
        lambda: M.kv_append(cache, k, k, slots, cos_t=table[:2], sin_t=table[:2]),
        lambda: M.kv_append(cache, k, k, slots, cos_t=table, sin_t=table, col0=50),
        lambda: M.KVCache(cache.k, cache.v[:1]), lambda: M.KVCache(cache.k.float(), cache.v.float()),
        lambda: M.KVCache(cache.k, cache.v, k_scales=torch.zeros(2, 2, 16, 2, dtype=torch.uint8, device="cuda")),
        lambda: M.KVCache(cache.k.transpose(1, 2), cache.v.transpose(1, 2)),
        lambda: M.kv_append(M.KVCache(cache.k[:, :, :8].contiguous(), cache.v[:, :, :8].contiguous()), k, k, slots),
        lambda: M.kv_append(M.KVCache(cache.k[..., :48].contiguous(), cache.v[..., :48].contiguous()), k[..., :48], k[..., :48], slots),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((M.MRError, TypeError, ValueError)):
            call()
            print("accepted", i)
