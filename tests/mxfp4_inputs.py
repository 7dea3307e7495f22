"""Plain numpy forms of the MXFP4 and routed-expert operators, in 64 bits.

Test infrastructure.  bf16 tensors are uint16 bit arrays, packed words uint32,
scales uint8.
"""
from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
BF16_ROUND, F32_ROUND = 2.0 ** -8, 2.0 ** -24  # a rounding's error is at most half a step


def to_bf16(x):
    """float32 -> bf16 bits, to nearest even (finite values and infinities)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    nan = np.isnan(np.asarray(x, np.float32))
    return np.where(nan, np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.ascontiguousarray(b).astype(np.uint32) << 16).view(np.float32)


def power(byte):
    """2^(byte - 127) in 64 bits, NaN at 255."""
    b = np.asarray(byte).astype(np.float64)
    return np.where(b == 255, np.nan, np.exp2(b - 127))


def quantize(x):
    """(packed uint32 [rows, cols / 8], scales uint8 [rows, cols / 32]) of a
    float32 [rows, cols], by distance to every e2m1 number."""
    b = np.asarray(x, np.float32).reshape(x.shape[0], -1, 32)
    finite = np.isfinite(b).all(-1)
    v = np.where(finite[..., None], b, 0).astype(np.float64)
    top = np.abs(v).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1))), -1e9)
    # log2 may round up to a whole number just below it
    e = np.where((top > 0) & (np.exp2(np.clip(e, -1074, 1023)) > top), e - 1, e)
    byte = np.clip(e - 2 + 127, 0, 254)
    m = np.abs(v) / np.exp2(byte - 127)[..., None]
    d = np.abs(m[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(near.sum(-1) > 1, even.argmax(-1), near.argmax(-1))
    code = code + 8 * np.signbit(b)
    code = np.where(finite[..., None], code, 0).astype(np.uint32)
    words = (code.reshape(x.shape[0], -1, 8) << (4 * np.arange(8, dtype=np.uint32))).sum(-1).astype(np.uint32)
    return words, np.where(finite, byte, 255).astype(np.uint8)


def values(packed, scales):
    """float64 [..., cols] of words [..., cols / 8] and bytes [..., cols / 32]."""
    code = (packed[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    v = GRID[code & 7] * np.where(code >= 8, -1.0, 1.0)
    v = v.reshape(*scales.shape, 32) * power(scales)[..., None]
    return v.reshape(*packed.shape[:-1], -1)


def matrix(rng, rows, cols, lead=(), std=1.0, lo=None, hi=None):
    """A random MXFP4 matrix: any codes, and scales of a few octaves round
    those of values of standard deviation std (or bytes lo .. hi - 1)."""
    packed = rng.integers(0, 2 ** 32, (*lead, rows, cols // 8), dtype=np.uint64).astype(np.uint32)
    mid = int(np.floor(np.log2(std))) + 126
    scales = rng.integers(mid - 2 if lo is None else lo, mid + 2 if hi is None else hi, (*lead, rows, cols // 32))
    return packed, scales.astype(np.uint8)


def order(ids, experts):
    """(offsets, pair_of_row, row_of_pair) by walking the pairs."""
    lists = [[] for _ in range(experts)]
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < experts:
            lists[e].append(p)
    rows = [p for of in lists for p in of]
    row_of_pair = np.full(ids.size, -1, np.int32)
    row_of_pair[rows] = np.arange(len(rows))
    offsets = np.cumsum([0] + [len(of) for of in lists]).astype(np.int32)
    pair_of_row = np.full(ids.size, -1, np.int32)
    pair_of_row[:len(rows)] = rows
    return offsets, pair_of_row, row_of_pair.reshape(ids.shape)


def ids_of(rng, tokens, per_token, experts, kind):
    """Expert ids: `spread`, `hot` (half of the slots on one expert), `one` (all
    on the last), `dropped` (a third outside, on both sides), `none` (all
    outside), `twice` (a token may name an expert more than once)."""
    if kind == "one":
        return np.full((tokens, per_token), experts - 1, np.int32)
    if kind == "none":
        return np.where(rng.random((tokens, per_token)) < 0.5, -1, experts).astype(np.int32)
    if kind == "twice":
        return rng.integers(0, max(1, experts // 4), (tokens, per_token)).astype(np.int32)
    if per_token <= experts:
        ids = np.argsort(rng.random((tokens, experts)), axis=1)[:, :per_token].astype(np.int32)
    else:
        ids = rng.integers(0, experts, (tokens, per_token)).astype(np.int32)
    if kind == "hot":
        ids = np.where(rng.random(ids.shape) < 0.5, experts // 2, ids)
    if kind == "dropped":
        out = rng.random(ids.shape)
        ids = np.where(out < 0.17, -1 - ids, np.where(out < 0.34, ids + experts, ids))
    return ids.astype(np.int32)


def dev(a):
    import torch

    a = np.ascontiguousarray(a)
    t = torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a.view(np.int16) if a.dtype == np.uint16 else a)
    return (t.view(torch.bfloat16) if a.dtype == np.uint16 else t).cuda()


def host(t):
    """A tensor as float64 (bf16 and f32) or as its integers."""
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()
