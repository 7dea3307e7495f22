"""Appended keys whose way to the stored value leaves f32's range while the value itself does
not: products that fall below it before a large weight, and sums that pass its largest value.
What is stored is compared bit for bit with 64 bits (test_gpu_kv_append.py)."""
import numpy as np
import pytest

import kv_inputs as K
import mxfp4_inputs as X
from test_gpu_kv_append import expect, stored

pytestmark = pytest.mark.gpu
EPS = float(np.float32(1e-6))


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def check(M, rng, x, mxfp4, w=None, cos=None, sin=None, halves=False):
    """Appends x [tokens, heads, dim] f32 as keys and values."""
    T, H, D = x.shape
    pages = K.Pages(rng, -(-T // 16) + 1, H, 16, D, mxfp4)
    cache = pages.device(M)
    slots = rng.permutation(pages.shape[0] * 16)[:T].astype(np.int32)
    k64, how = x.astype(np.float64), {}
    if w is not None:
        k64 = K.norm(k64, w.astype(np.float64), EPS)
        how.update(normalize=True, norm_weight=X.dev(w), eps=EPS)
    if cos is not None:
        k64 = K.turn(k64, cos, sin, 0, halves)
        how.update(cos_t=X.dev(cos), sin_t=X.dev(sin), halves=halves)
    M.kv_append(cache, X.dev(x), X.dev(x), X.dev(slots), **how)
    with np.errstate(over="ignore"):
        want = expect(pages, k64, x.astype(np.float64), slots)
    for name, a, b in zip(("k", "v", "k_scales", "v_scales"), stored(cache), want):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:3])


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("low,weight", [(-80, 60), (-95, 30), (-105, 30), (-105, 60), (-120, 60), (-125, 100), (-140, 120)])
def test_small_values_under_large_weights(M, low, weight, rotated, mxfp4):
    """Beside a block of values around 2^40, so that x / norm is about 2^(low - 40): below f32's normal
    numbers, or all of them.  (Of one sign: -0 is told from 0.)"""
    rng = np.random.default_rng([-low, weight])
    T, H, D = 24, 2, 128
    x = rng.uniform(0.5, 2, (T, H, D)).astype(np.float32) * np.float32(2.0 ** low)
    x[..., :32] = 2.0 ** 40 * rng.uniform(0.5, 2, (T, H, 32))
    x[..., 70] = 0
    w = np.full(D, 2.0 ** weight, np.float32)
    w[:32] = 1
    cos, sin = (np.abs(t) for t in K.tables(rng, T, D // 2)) if rotated else (None, None)
    check(M, rng, x, mxfp4, w, cos, None if sin is None else 1e-3 * sin)


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("halves", [False, True])
def test_rotations_past_the_largest_f32(M, halves, mxfp4):
    """Both of a pair near 3.4e38, turned by 45 degrees: 4.8e38 is past f32 and bf16, not past MXFP4."""
    rng = np.random.default_rng(4)
    T, H, D = 40, 2, 128
    x = (rng.uniform(0.3, 1.0, (T, H, D)) * 3.4e38).astype(np.float32) * rng.choice([-1, 1], (T, H, D)).astype(np.float32)
    x[::3, :, 32:64] *= np.float32(1e-3)  # (blocks on either side)
    x[1::3, :, 64:] *= np.float32(1e-30)
    angle = rng.choice([0.25, 0.75, -0.25, 1.25, 0.1], (T, D // 2)) * np.pi
    check(M, rng, x, mxfp4, None, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32), halves)


@pytest.mark.parametrize("mxfp4", [False, True])
@pytest.mark.parametrize("rotated", [False, True])
def test_weights_near_the_largest_f32(M, rotated, mxfp4):
    """A normalised value of up to sqrt(dim) times the largest weight: past every power of a block, which keeps 6 of the last."""
    rng = np.random.default_rng(6)
    T, H, D = 24, 1, 128
    x = rng.standard_normal((T, H, D)).astype(np.float32)
    x[::2, :, 5] = 1e4
    w = (rng.uniform(0.2, 1.0, D) * 3.4e38).astype(np.float32)
    w[96:] = 1
    cos, sin = K.tables(rng, T, D // 2) if rotated else (None, None)
    check(M, rng, x, mxfp4, w, cos, sin, True)
