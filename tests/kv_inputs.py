"""Plain numpy forms of the head norms, the cache appends and the attention over
pages, in 64 bits, and inputs for them.

Test infrastructure.  bf16 tensors are uint16 bit arrays.
"""
from __future__ import annotations

import numpy as np

import mxfp4_inputs as X

U = X.F32_ROUND  # 2^-24
MFMA = 2.0 ** -23  # a matrix instruction's sums are cut off, not rounded


def values_of(rng, shape, f32, std=1.0):
    """(device tensor, the same in 64 bits)."""
    x = (std * rng.standard_normal(shape)).astype(np.float32)
    if f32:
        return X.dev(x), x.astype(np.float64)
    b = X.to_bf16(x)
    return X.dev(b), X.from_bf16(b).astype(np.float64)


def tables(rng, rows, half):
    """cos, sin f32 of random angles."""
    a = rng.uniform(-4, 4, (rows, half))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def turn(x, cos, sin, col0, halves, inverse=False):
    """x [tokens, heads, dim] with columns col0 .. rotated; cos, sin [tokens, n]."""
    y, n = x.copy(), cos.shape[1]
    for i in range(n):
        a, b = (col0 + i, col0 + i + n) if halves else (col0 + 2 * i, col0 + 2 * i + 1)
        c, s = cos[:, None, i].astype(np.float64), sin[:, None, i].astype(np.float64) * (-1 if inverse else 1)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def spread(x, cos, sin, col0, halves):
    """The sum of the magnitudes that a rotation adds up, for |x|."""
    return turn(np.abs(x), np.abs(cos), -np.abs(sin), col0, halves) if not x.size else np.maximum(
        turn(np.abs(x), np.abs(cos), np.abs(sin), col0, halves), turn(np.abs(x), np.abs(cos), -np.abs(sin), col0, halves))


def norm(x, w, eps):
    r = 1 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    return w * (x * r)


def norm_backward(dy, x, w, eps, cos, sin, col0, halves):
    """(dx, dw, a bound of dx's terms, the sum of |terms| of dw)."""
    g = turn(dy, cos, sin, col0, halves, inverse=True)
    around = spread(dy, cos, sin, col0, halves)
    r = 1 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    unit = x * r
    dw, dw_sum = (g * unit).sum((0, 1)), (around * np.abs(unit)).sum((0, 1))
    gw = g * w
    dot = (gw * unit).mean(-1, keepdims=True)
    dot_sum = (around * np.abs(w * unit)).mean(-1, keepdims=True)
    return r * (gw - unit * dot), dw, r * (15 * around * np.abs(w) + 54 * np.abs(unit) * dot_sum), dw_sum


def round_bf16(x):
    """64 bits to bf16 (uint16), once, to nearest even."""
    m, e = np.frexp(np.where(np.isfinite(x), x, 0))
    step = np.maximum(e - 8, -133)  # (below 2^-126 a bf16's steps are 2^-133)
    y = np.ldexp(np.rint(np.ldexp(m, e - step)), step).astype(np.float32)
    return X.to_bf16(np.where(np.isfinite(x), y, x).astype(np.float32))


def quantize64(x):
    """mxfp4_inputs.quantize for 64-bit values [rows, cols]."""
    b = x.reshape(x.shape[0], -1, 32)
    finite = np.isfinite(b).all(-1)
    v = np.where(finite[..., None], b, 0)
    top = np.abs(v).max(-1)
    byte = np.clip(np.where(top > 0, np.frexp(top)[1] - 1, -1000) - 2 + 127, 0, 254)
    m = np.abs(v) / np.exp2(byte - 127.0)[..., None]
    d = np.abs(m[..., None] - X.GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(near.sum(-1) > 1, even.argmax(-1), near.argmax(-1)) + 8 * np.signbit(b)
    code = np.where(finite[..., None], code, 0).astype(np.uint32)
    words = (code.reshape(x.shape[0], -1, 8) << (4 * np.arange(8, dtype=np.uint32))).sum(-1).astype(np.uint32)
    return words, np.where(finite, byte, 255).astype(np.uint8)


class Pages:
    """A cache's pages on the host: random rows, also where no sequence has any."""

    def __init__(self, rng, pages, heads, page_size, dim, mxfp4, std=1.0):
        self.mxfp4, self.shape = mxfp4, (pages, heads, page_size, dim)
        if mxfp4:
            parts = [X.matrix(rng, heads * page_size, dim, (pages,), std) for _ in range(2)]
            self.k, self.v = (p[0].reshape(*self.shape[:3], dim // 8) for p in parts)
            self.ks, self.vs = (p[1].reshape(*self.shape[:3], dim // 32) for p in parts)
        else:
            self.k, self.v = (X.to_bf16((std * rng.standard_normal(self.shape)).astype(np.float32)) for _ in range(2))
            self.ks = self.vs = None

    def values(self):
        """(keys, values) [pages, heads, page_size, dim] in 64 bits; MXFP4 values past
        the largest bf16 are infinite, as dequantized."""
        if self.mxfp4:
            both = X.values(self.k, self.ks), X.values(self.v, self.vs)
            return tuple(np.where(np.abs(x) >= 2.0 ** 128, np.copysign(np.inf, x), x) for x in both)
        return X.from_bf16(self.k).astype(np.float64), X.from_bf16(self.v).astype(np.float64)

    def device(self, M, gap=0):
        """The cache on the GPU; gap: pages that many elements (a multiple of 16 bytes) further apart."""
        import torch

        def put(a, extra):
            t = X.dev(a)
            if not extra:
                return t
            flat = t.reshape(t.shape[0], -1)
            wide = torch.zeros(t.shape[0], flat.shape[1] + extra, dtype=t.dtype, device="cuda")
            wide[:, :flat.shape[1]] = flat
            return wide[:, :flat.shape[1]].unflatten(1, t.shape[1:])

        if self.mxfp4:
            return M.KVCache(put(self.k, gap), put(self.v, gap), put(self.ks, gap), put(self.vs, gap))
        return M.KVCache(put(self.k, gap), put(self.v, gap))


def page_tables(rng, lens, page_size, spare=2, pad=-7):
    """(table int32 [batch, most], pages): pages in any order, `pad` behind a sequence's last."""
    need = [-(-n // page_size) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table, at = np.full((len(lens), max(need + [1])), pad, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def attention(q, k, v, table, lens, offsets, scale, window=0, sinks=None):
    """(out, lse, the sum of p |v|, the largest sum of |q k| scale) in 64 bits: q
    [tokens, heads, dim]; k, v [pages, kv_heads, page_size, dim]."""
    T, H, D = q.shape
    pages, kvh, ps, _ = k.shape
    out, lse = np.full(q.shape, np.nan), np.full((T, H), np.nan)
    weight, terms = np.zeros(q.shape), np.zeros((T, H))
    for b, n in enumerate(lens):
        q0, q1 = (b, b + 1) if offsets is None else (int(offsets[b]), int(offsets[b + 1]))
        ids = table[b, :-(-n // ps)]
        there = np.repeat((ids >= 0) & (ids < pages), ps)[:n]
        rows = [np.moveaxis(a[np.clip(ids, 0, max(pages - 1, 0))], 1, 0).reshape(kvh, -1, D)[:, :n] for a in (k, v)]
        for t in range(q0, q1):
            pos = n - (q1 - q0) + (t - q0)
            seen = there & (np.arange(n) <= pos)
            if window:
                seen &= np.arange(n) > pos - window
            for h in range(H):
                kk, vv = rows[0][h * kvh // H][seen], rows[1][h * kvh // H][seen]
                s = kk @ q[t, h] * scale
                every = s if sinks is None else np.append(s, sinks[h])
                if not len(s) and (sinks is None):
                    out[t, h], lse[t, h] = 0, -np.inf
                    continue
                top = every.max()
                total = np.exp(every - top).sum()
                p = np.exp(s - top) / total
                out[t, h], lse[t, h] = p @ vv, top + np.log(total)
                weight[t, h] = p @ np.abs(vv)
                terms[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max(initial=0) * scale
    return out, lse, weight, terms
