"""Products with MXFP4 weights whose scale bytes are 253 and 254.

Taken in bf16, a weight of at least 2^128 is infinite: times an activation
that is not zero it gives an infinity of the product's sign, times zero NaN, as
in IEEE arithmetic, whatever the activation's type and bits.  Activations in
MXFP4 meet the stored numbers, which are finite.

One weight of a row is large, the others are small whole numbers (and halves),
and so are the activations.  Where the large weight's code is zero, a row's sum is
below 2^21 and exact in any order.  Otherwise it is L + s, L the large product and
|s| < 2^-100 |L|, in n f32 additions.  The matrix instructions do not round to the
nearest: 2^127 - 315 came out as the number below 2^127, which is 2^103 away.  An
addition that cuts off what lies below the last bit is off by less than one step, at
most 2^-23 of the sum, and a sum to the nearest by half of one: |error| <= n 2^-23
|L| (1.001 for the growth of L with the errors).  A sum is an infinity only from (1 -
2^-25) 2^128 less such an error on.  Infinities and NaN of infinite weights have to be
where they are in the sums of the definition."""
import numpy as np
import pytest

import mxfp4_inputs as X

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f32", "mxfp4"]


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


def large_weights(rng, rows, cols, lead=()):
    """Packed words, bytes and the values in 64 bits: row o has a block of byte 253 or
    254 whose only code that is not zero runs over all sixteen."""
    packed, scales = X.matrix(rng, rows, cols, lead, lo=126, hi=129)
    codes = ((packed[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(*lead, rows, cols)
    at = rng.integers(0, cols, (*lead, rows))
    for i in np.ndindex(*lead, rows):
        c = at[i]
        codes[i][c // 32 * 32:c // 32 * 32 + 32] = 0
        codes[i][c] = i[-1] % 16
        scales[i][c // 32] = 253 + i[-1] // 16 % 2
    packed = (codes.reshape(*lead, rows, cols // 8, 8).astype(np.uint32) << (4 * np.arange(8, dtype=np.uint32))).sum(-1)
    packed = packed.astype(np.uint32)
    return packed, scales, X.values(packed, scales)


def activations(rng, kind, rows, cols):
    """Whole numbers other than zero, zeros in every third row only; MXFP4: scales of
    2^-30, for products that stay finite."""
    if kind == "mxfp4":
        packed, scales = X.matrix(rng, rows, cols, lo=97, hi=98)
        return (packed, scales), X.values(packed, scales)
    x = rng.integers(1, 8, (rows, cols)) * rng.choice([-1.0, 1.0], (rows, cols))
    if rows > 2:
        x[2::3][rng.random(x[2::3].shape) < 0.3] = 0
    x = x.astype(np.float32)
    return (x if kind == "f32" else X.to_bf16(x)), x.astype(np.float64)


def product(kind, x64, w64):
    """The sums in 64 bits, and the largest |product| of each where it is large."""
    w = w64 if kind == "mxfp4" else np.where(np.abs(w64) >= 2.0 ** 128, np.copysign(np.inf, w64), w64)
    large = np.abs(w) >= 2.0 ** 100
    at = large.argmax(1)  # the large weight, where there is one
    big = np.where(large.any(1), w[np.arange(len(w)), at], 0)
    with np.errstate(invalid="ignore"):
        top = np.where(big == 0, 0, x64[:, at] * np.where(big == 0, 1, big))
    return x64 @ np.where(large, 0, w).T + top, np.abs(top)


def operand(M, x):
    return M.MXFP4Weights(X.dev(x[0]), X.dev(x[1])) if isinstance(x, tuple) else X.dev(x)


def check(got, want, top, terms, what):
    """`terms`: additions of a sum."""
    got = X.host(got)
    rel = 1.001 * terms * 2.0 ** -23
    with np.errstate(invalid="ignore"):
        ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.isfinite(want) & (np.abs(got - want) <= rel * top))
        ok |= np.isfinite(want) & (got == np.copysign(np.inf, want)) & (np.abs(want) >= 2.0 ** 128 * (1 - 2.0 ** -25) * (1 - rel))
    assert ok.all(), (what, int((~ok).sum()), got[~ok][:8], want[~ok][:8])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,out,inp", [(1, 70, 96), (2, 300, 544), (5, 70, 288), (16, 264, 1056), (40, 70, 2080), (70, 520, 96),
                                            (100, 4104, 288), (100, 8200, 288), (300, 16392, 288), (600, 16392, 256)])
def test_infinite_weights(M, tokens, out, inp, kind):
    import torch

    rng = np.random.default_rng(tokens + out)
    packed, scales, w64 = large_weights(rng, out, inp)
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    x, x64 = activations(rng, kind, tokens, inp)
    want, top = product(kind, x64, w64)
    assert kind == "mxfp4" or np.isinf(want).any()
    check(M.mxfp4_mm(operand(M, x), w, out_dtype=torch.float32), want, top, inp * (3 if kind == "f32" else 1), (tokens, out, inp))


def test_f32_activations_of_every_length(M):
    # 1 to 24 significant bits, and powers of two over the range whose first part
    # is not zero, against weights that are infinite and against 3 2^126
    import torch

    bits = [np.float32(1 + (1 - 2.0 ** -n)) for n in range(24)]
    powers = [np.float32(2.0 ** e) for e in (-133, -126, -100, -1, 0, 1, 100, 127)]
    x = np.zeros((len(bits) + len(powers), 32), np.float32)
    x[:, 7] = np.array(bits + powers) * np.tile([1, -1], len(x) // 2)
    for code, byte in ((7, 254), (15, 254), (6, 253), (4, 254), (5, 253)):
        packed = np.zeros((20, 4), np.uint32)
        packed[:, 0] = code << 28
        value = X.values(packed, np.full((20, 1), byte, np.uint8))[0, 7]
        value = np.copysign(np.inf, value) if abs(value) >= 2.0 ** 128 else value
        want = np.repeat((x[:, 7].astype(np.float64) * value)[:, None], 20, 1)
        w = M.MXFP4Weights(X.dev(packed), X.dev(np.full((20, 1), byte, np.uint8)))
        check(M.mxfp4_mm(X.dev(x), w), want, np.abs(want), 3, (code, byte))


@pytest.mark.parametrize("by_row", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,per_token,experts,out,inp", [(1, 4, 8, 70, 96), (40, 3, 9, 160, 288), (200, 8, 16, 520, 160),
                                                              (300, 8, 60, 600, 288), (500, 8, 20, 392, 256)])
def test_infinite_expert_weights(M, tokens, per_token, experts, out, inp, kind, by_row):
    import torch

    rng = np.random.default_rng(tokens + out)
    ids = X.ids_of(rng, tokens, per_token, experts, "spread")
    offsets, pair, _ = X.order(ids, experts)
    packed, scales, w64 = large_weights(rng, out, inp, (experts,))
    w = M.MXFP4Weights(X.dev(packed), X.dev(scales))
    x, x64 = activations(rng, kind, tokens * per_token if by_row else tokens, inp)
    want, top = np.zeros((tokens * per_token, out)), np.zeros((tokens * per_token, out))
    for e in range(experts):
        r = np.arange(offsets[e], offsets[e + 1])
        if r.size:
            want[r], top[r] = product(kind, x64[r if by_row else pair[r] // per_token], w64[e])
    o = M.expert_sort(X.dev(ids), experts)
    check(M.mxfp4_expert_mm(operand(M, x), w, o, sorted_rows=by_row, out_dtype=torch.float32), want, top,
          inp * (3 if kind == "f32" else 1), by_row)
