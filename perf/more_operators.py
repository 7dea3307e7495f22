"""The operators of grouped-query attention over a paged key/value cache,
measured: the calls that a program makes of them, over the sizes it makes them
with.

    listed()            the cases looked at one by one
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what the program holds before the call (on the GPU)
    run(state)          one pass; returns its outputs whole
    work(case)          the bytes and flops a pass cannot do without
    exact(case, seed)   the outputs in 64 bits, from the definitions

Kinds ("op"):
    norm     RMSNorm of every head of the queries and keys, and the rotation by
             their positions, in one pass: "forward", and "backward" with the
             gradients of the inputs and of the two weights
    append   keys (normalised and rotated on the way) and values into the pages
             of a cache that holds bf16 or MXFP4
    attend   attention of one or more queries of each sequence over such a
             cache, a page table and lengths

`own` false: plain torch in 32 bits (64 for what is rounded to 4 bits); true:
the library's calls.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1
_EPS = 1e-6


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minirun-app_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import minirun_hip

    return minirun_hip


# ---------------------------------------------------------------- the cases
def _norm(direction, tokens, heads, kv_heads, dim, rope, col0, halves, dtype):
    return {"op": "norm", "direction": direction, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rope": rope, "col0": col0, "halves": halves, "dtype": dtype}


def _append(tokens, kv_heads, dim, page, cache, norm, rope, halves, dtype):
    return {"op": "append", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "norm": norm,
            "rope": rope, "halves": halves, "dtype": dtype}


def _attend(batch, queries, keys, spread, heads, kv_heads, dim, page, cache, window=0, sinks=False):
    return {"op": "attend", "batch": batch, "queries": queries, "keys": keys, "spread": spread, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "window": window, "sinks": sinks}


def listed():
    return [
        # one decode step of one sequence: launches are all of it
        {"name": "norm_t1_h32_4", **_norm("forward", 1, 32, 4, 128, 128, 0, True, "bf16")},
        # a prompt's queries and keys
        {"name": "norm_t4096_h32_4", **_norm("forward", 4096, 32, 4, 128, 128, 0, True, "bf16")},
        # the gradients of a training batch of 8192 tokens
        {"name": "norm_t8192_h32_8_backward", **_norm("backward", 8192, 32, 8, 128, 128, 0, True, "bf16")},
        # an odd number of tokens in f32, heads whose tail alone is rotated, as adjacent pairs
        {"name": "norm_t777_h12_2_d96_f32_backward", **_norm("backward", 777, 12, 2, 96, 64, 32, False, "f32")},
        # the new tokens of 32 sequences' decode step, into 4 bits
        {"name": "append_t32_mxfp4", **_append(32, 4, 128, 16, "mxfp4", True, 128, True, "bf16")},
        # a prompt's keys and values, into 4 bits
        {"name": "append_t8192_mxfp4", **_append(8192, 8, 128, 64, "mxfp4", True, 128, True, "bf16")},
        # the same into bf16 pages, keys rotated only
        {"name": "append_t4001_bf16", **_append(4001, 8, 128, 32, "bf16", False, 128, True, "bf16")},
        # a short chat's next token: latency
        {"name": "attend_b1_n500", **_attend(1, 1, 500, 1.0, 32, 4, 128, 16, "mxfp4")},
        # a serving batch, sequences of 1000 to 12000 tokens
        {"name": "attend_b64_n12000", **_attend(64, 1, 12000, 12.0, 32, 4, 128, 32, "mxfp4")},
        # one long document
        {"name": "attend_b1_n131072", **_attend(1, 1, 131072, 1.0, 64, 8, 128, 64, "mxfp4")},
        # five drafted tokens to check in each of eight sequences, bf16 pages, the last 4096 positions only
        {"name": "attend_b8_q5_n9000_window_bf16", **_attend(8, 5, 9000, 3.0, 32, 8, 128, 16, "bf16", 4096, True)},
        # a prompt chunk of 4096 tokens behind 1000 cached ones
        {"name": "attend_q4096_n5096", **_attend(1, 4096, 5096, 1.0, 32, 4, 128, 64, "mxfp4")},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "attend", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 8])
    if op == "norm":
        dim = rng.choice([64, 96, 128, 128, 256, 512, 2 * rng.randint(16, 256)])
        heads = kv * rng.choice([1, 3, 4, 8])
        rope = rng.choice([dim, 2 * (dim // 4), 2 * rng.randint(1, dim // 2)])
        return _norm(rng.choice(["forward", "backward"]), _log(rng, 1, max(1, min(8192, 20_000_000 // (dim * (heads + kv))))),
                     heads, kv, dim, rope, rng.choice([0, dim - rope]), rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"]))
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    page, cache = rng.choice([16, 32, 48, 64, 128]), rng.choice(["mxfp4", "mxfp4", "bf16"])
    if op == "append":
        return _append(_log(rng, 1, 8_000_000 // (dim * kv)), kv, dim, page, cache, rng.random() < 0.5,
                       rng.choice([0, dim, dim // 2]), rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"]))
    group = rng.choice([1, 2, 4, 5, 7, 8, 16])
    queries = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 4096)])
    # at most 150 MB of cache and 2e11 operations
    most = 50_000_000_000 // (queries * kv * group * dim)
    keys = min(queries + _log(rng, 1, 60_000) - 1, max(queries, most))
    if keys > most:  # (the longest prompts of many heads)
        queries = keys = math.isqrt(most * queries)
    batch = _log(rng, 1, max(1, min(64, 75_000_000 // (keys * kv * (2 * dim if cache == "bf16" else dim // 2 + dim // 32)),
                                    most // keys, 30_000_000 // (queries * kv * group * dim))))
    return _attend(batch, queries, keys, rng.choice([1.0, 4.0, 100.0]), kv * group, kv, dim, page, cache,
                   rng.choice([0, 0, 0, _log(rng, 16, 8192)]), rng.random() < 0.25)


# ---------------------------------------------------------------- plain MXFP4
def _codes(x):
    """Codes (0..15) and scale bytes of the blocks of 32 of x (f64), int32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1)
    byte = torch.where(top > 0, torch.frexp(top).exponent.double() + (126 - 2), 0.0).clamp(0, 254)
    m = b.abs() * torch.exp2(127 - byte)[..., None]
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int()
            + (m >= 3.5).int() + (m > 5.0).int())
    return (code + 8 * torch.signbit(b).int()).reshape(x.shape), byte.int()


def _pack(code):
    c = code.reshape(*code.shape[:-1], -1, 8)
    word = c[..., 0].clone()
    for j in range(1, 8):
        word |= c[..., j] << (4 * j)
    return word


def _values(packed, scales):
    """f32 [..., dim] of words [..., dim / 8] and bytes [..., dim / 32]."""
    shift = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
    code = (packed[..., None] >> shift) & 15
    table = torch.tensor(_GRID + tuple(-g for g in _GRID), device=packed.device)
    power = torch.exp2(scales.float() - 127)
    return (table[code.long()].reshape(*scales.shape, 32) * power[..., None]).reshape(*packed.shape[:-1], -1)


# ---------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return (std * torch.randn(*shape, generator=self.g, device="cuda")).to(dtype)

    def whole(self, n, hi):
        return torch.randint(0, hi, (n,), generator=self.g, device="cuda")

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def heads(self, tokens, heads, dim, dtype):
        """A projection's rows: heads of their own size each, a few large features."""
        x = self.normal(tokens, heads, dim, dtype=torch.float32)
        x *= torch.exp(0.5 * torch.randn(1, heads, 1, generator=self.g, device="cuda"))
        x *= torch.where(torch.rand(1, 1, dim, generator=self.g, device="cuda") < 0.02, 8.0, 1.0)
        return x.to(dtype)

    def weight(self, dim, dtype):
        return (1 + 0.1 * torch.randn(dim, generator=self.g, device="cuda")).to(dtype)


def _tables(rows, rope):
    """cos and sin f32 [rows, rope / 2] of the angles position * 10000^(-2 i / rope)."""
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * torch.exp(
        torch.arange(0, rope, 2, device="cuda", dtype=torch.float64) * (-math.log(10000.0) / max(rope, 1)))
    return torch.cos(angle).float(), torch.sin(angle).float()


def _lengths(case):
    """Keys of each sequence, the longest first: spread 12 ends at a twelfth of it."""
    B, n, q = case["batch"], case["keys"], case["queries"]
    return [max(q, round(n * case["spread"] ** (-i / (B - 1)))) if B > 1 else n for i in range(B)]


def prepare(case, seed):
    r, op = _Rand(seed), case["op"]
    st = {"op": op, "case": dict(case)}
    if op == "norm":
        T, D, dt = case["tokens"], case["dim"], _DT[case["dtype"]]
        st["q"], st["k"] = r.heads(T, case["heads"], D, dt), r.heads(T, case["kv_heads"], D, dt)
        st["wq"], st["wk"] = r.weight(D, dt), r.weight(D, dt)
        st["cos"], st["sin"] = _tables(max(T, 4096), case["rope"])
        st["positions"] = ((torch.arange(T, device="cuda") + r.whole(1, 4096)) % max(T, 4096)).int()
        if case["direction"] == "backward":
            st["dq"], st["dk"] = r.normal(*st["q"].shape, dtype=dt), r.normal(*st["k"].shape, dtype=dt)
        return st
    H, D, page = case["kv_heads"], case["dim"], case["page"]
    if op == "append":
        T, dt = case["tokens"], _DT[case["dtype"]]
        pages = -(-T // page) + 1
        st["k"], st["v"] = r.heads(T, H, D, dt), r.heads(T, H, D, dt)
        st["weight"] = r.weight(D, dt) if case["norm"] else None
        st["cos"], st["sin"] = _tables(max(T, 4096), case["rope"]) if case["rope"] else (None, None)
        st["positions"] = ((torch.arange(T, device="cuda") + r.whole(1, 4096)) % max(T, 4096)).int()
        # the rows of consecutive tokens in pages of any order; one token in 64 is padding
        st["slots"] = (r.order(pages)[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:T].int()
        st["slots"] = torch.where(r.whole(T, 64) == 0, -1, st["slots"]) if T > 1 else st["slots"]
    else:
        lens, q = _lengths(case), case["queries"]
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        st["q"] = r.normal(case["batch"] * q, case["heads"], D, std=1.5)
        st["scale"] = D ** -0.5
        order, table, at = r.order(pages), torch.full((case["batch"], max(need)), -1, device="cuda"), 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        st["table"], st["lens"] = table.int(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        st["offsets"] = (torch.arange(case["batch"] + 1, device="cuda") * q).int() if q > 1 else None
        st["sinks"] = r.normal(case["heads"], dtype=torch.float32) if case["sinks"] else None
    shape = (pages, H, page, D)
    if case["cache"] == "bf16":
        st["cache"] = (r.normal(*shape), r.normal(*shape))
    else:
        parts = []
        for _ in range(2):
            words = torch.empty(*shape[:-1], D // 8, dtype=torch.int32, device="cuda")
            scales = torch.empty(*shape[:-1], D // 32, dtype=torch.uint8, device="cuda")
            for lo in range(0, pages, 256):  # (in pieces: the 64-bit form is large)
                code, byte = _codes(r.normal(min(256, pages - lo), *shape[1:], dtype=torch.float32).double())
                words[lo:lo + 256], scales[lo:lo + 256] = _pack(code), byte.to(torch.uint8)
            parts += [words, scales]
        st["cache"] = (parts[0], parts[2], parts[1], parts[3])
    if own:
        st["cache"] = _lib().KVCache(*st["cache"])
    return st


# ---------------------------------------------------------------- one pass
def _run_own(st):
    M = _lib()
    case = st["case"]
    if st["op"] == "norm":
        how = dict(q_weight=st["wq"], k_weight=st["wk"], eps=_EPS, cos_t=st["cos"], sin_t=st["sin"], positions=st["positions"],
                   col0=case["col0"], halves=case["halves"])
        if case["direction"] == "forward":
            return M.head_norm_rope(st["q"], st["k"], **how)
        return M.head_norm_rope_backward(st["dq"], st["q"], st["dk"], st["k"], **how)
    cache = st["cache"]
    if st["op"] == "attend":
        return M.kv_attention(st["q"], cache, st["table"], st["lens"], scale=st["scale"], q_offsets=st["offsets"],
                              window=case["window"], sinks=st["sinks"], max_kv_len=case["keys"])
    M.kv_append(cache, st["k"], st["v"], st["slots"], normalize=case["norm"], norm_weight=st["weight"], eps=_EPS,
                cos_t=st["cos"], sin_t=st["sin"], positions=st["positions"], halves=case["halves"])
    if case["cache"] == "bf16":
        return cache.k, cache.v
    return cache.values(torch.bfloat16)


def _turned(x, cos, sin, col0, halves, inverse=False):
    """Columns [col0, col0 + 2 n) of x [tokens, heads, dim] rotated by the angles of cos and sin [tokens, n]."""
    n = cos.shape[1]
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    if inverse:
        s = -s
    mid = x[..., col0:col0 + 2 * n]
    a, b = (mid[..., :n], mid[..., n:]) if halves else (mid[..., 0::2], mid[..., 1::2])
    ta, tb = a * c - b * s, a * s + b * c
    turned = torch.cat([ta, tb], -1) if halves else torch.stack([ta, tb], -1).flatten(-2)
    return torch.cat([x[..., :col0], turned, x[..., col0 + 2 * n:]], -1)


def _norm_plain(st):
    case, out, grads = st["case"], [], []
    at = st["positions"].long()
    cos, sin = st["cos"][at], st["sin"][at]
    for x, w, dy in ((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk"))):
        xf, wf = x.float(), w.float()
        inv = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + _EPS)
        if dy is None:
            out.append(_turned(xf * inv * wf, cos, sin, case["col0"], case["halves"]).to(x.dtype))
            continue
        g = _turned(dy.float(), cos, sin, case["col0"], case["halves"], inverse=True)
        unit = xf * inv
        grads.append((g * unit).sum((0, 1)))
        g = g * wf
        out.append((inv * (g - unit * (g * unit).mean(-1, keepdim=True))).to(x.dtype))
    return tuple(out + grads)


def _append_plain(st):
    case, cache, page = st["case"], st["cache"], st["case"]["page"]
    kept = (st["slots"] >= 0).nonzero()[:, 0]
    slots, at = st["slots"][kept].long(), st["positions"][kept].long()
    # what is rounded to 4 bits is computed in 64, next to a border
    k, v = st["k"][kept].double(), st["v"][kept].double()
    if case["norm"]:
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + _EPS) * st["weight"].double()
    if case["rope"]:
        k = _turned(k, st["cos"][at], st["sin"][at], 0, case["halves"])
    for i, x in enumerate((k, v)):
        if case["cache"] == "bf16":
            cache[i][slots // page, :, slots % page] = x.to(torch.bfloat16)
        else:
            code, byte = _codes(x)
            cache[i][slots // page, :, slots % page] = _pack(code)
            cache[2 + i][slots // page, :, slots % page] = byte.to(torch.uint8)
    if case["cache"] == "bf16":
        return cache[0], cache[1]
    return tuple(_values(cache[i], cache[2 + i]).to(torch.bfloat16) for i in (0, 1))


def _attend_plain(st):
    case, cache = st["case"], st["cache"]
    H, G, D, Q = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"], case["queries"]
    out = torch.empty_like(st["q"])
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - Q + 1 - case["window"]) // case["page"] if case["window"] else 0
        pages = st["table"][b, first:-(-n // case["page"])].long()
        parts = [c[pages] for c in cache]
        kv = [p.float() for p in parts] if case["cache"] == "bf16" else [_values(parts[i], parts[2 + i]) for i in (0, 1)]
        k, v = (x.transpose(0, 1).reshape(H, -1, D) for x in kv)
        where = first * case["page"] + torch.arange(k.shape[1], device=k.device)
        limit = n - Q + torch.arange(Q, device=k.device)[:, None]
        seen = where <= limit
        if case["window"]:
            seen &= where > limit - case["window"]
        for h in range(H):
            q = st["q"][b * Q:(b + 1) * Q, h * G:(h + 1) * G].float().reshape(Q * G, D)
            s = (q @ k[h].t()).reshape(Q, G, -1) * st["scale"]
            s = torch.where(seen[:, None], s, float("-inf"))
            top = s.amax(-1, keepdim=True)
            if st["sinks"] is not None:
                sink = st["sinks"][h * G:(h + 1) * G].reshape(1, G, 1)
                top = torch.maximum(top, sink)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            if st["sinks"] is not None:
                total = total + torch.exp(sink - top)
            o = (p.reshape(Q * G, -1) @ torch.where(seen.any(0)[:, None], v[h], 0.0)).reshape(Q, G, D) / total
            out[b * Q:(b + 1) * Q, h * G:(h + 1) * G] = o.to(out.dtype)
    return out


def _run_plain(st):
    return {"norm": _norm_plain, "append": _append_plain, "attend": _attend_plain}[st["op"]](st)


def run(st):
    return _run_own(st) if own else _run_plain(st)


# ---------------------------------------------------------------- minimal work
def _cache_bytes(case):
    """Bytes of one head's key or value."""
    return 2 * case["dim"] if case["cache"] == "bf16" else case["dim"] // 2 + case["dim"] // 32


def work(case):
    op, D = case["op"], case["dim"]
    if op == "norm":
        n, size = case["tokens"] * (case["heads"] + case["kv_heads"]) * D, 2 if case["dtype"] == "bf16" else 4
        tables = 4 * case["tokens"] * (case["rope"] + 1)
        forward = case["direction"] == "forward"
        return {"bytes": (2 if forward else 3) * size * n + tables, "flops": (6 if forward else 14) * n}
    if op == "append":
        n, size = case["tokens"] * case["kv_heads"] * 2, 2 if case["dtype"] == "bf16" else 4
        pages = -(-case["tokens"] // case["page"]) + 1
        whole = pages * case["page"] * case["kv_heads"] * 2
        # the new rows in and out, and for 4 bits the cache's values, which are returned
        read_back = whole * (_cache_bytes(case) + 2 * D) if case["cache"] == "mxfp4" else 0
        return {"bytes": n * (size * D + _cache_bytes(case)) + read_back + 4 * case["tokens"] * (case["rope"] + 2),
                "flops": 8 * n * D}
    keys = pairs = 0
    for n in _lengths(case):
        w, Q = case["window"] or n, case["queries"]
        keys += min(n, w + Q - 1)
        pairs += sum(min(n - Q + i + 1, w) for i in range(Q))
    rows = case["batch"] * case["queries"] * case["heads"]
    return {"bytes": 2 * keys * case["kv_heads"] * _cache_bytes(case) + 4 * rows * D, "flops": 4 * pairs * case["heads"] * D}


# ---------------------------------------------------------------- 64 bits
def _matrices64(cos, sin, halves):
    """Rotation matrices [tokens, 2 n, 2 n] of the pairs of columns."""
    T, n = cos.shape
    m = torch.zeros(T, 2 * n, 2 * n, dtype=torch.float64, device=cos.device)
    i = torch.arange(n, device=cos.device)
    a, b = (i, i + n) if halves else (2 * i, 2 * i + 1)
    m[:, a, a] = m[:, b, b] = cos.double()
    m[:, a, b], m[:, b, a] = -sin.double(), sin.double()
    return m


def _norm64(st, case):
    D, lo, hi = case["dim"], case["col0"], case["col0"] + case["rope"]
    ys = [[], []]
    grads = [torch.zeros(D, dtype=torch.float64, device="cuda") for _ in range(2)]
    step = max(1, 20_000_000 // (case["rope"] ** 2))
    for t in range(0, case["tokens"], step):
        at = st["positions"][t:t + step].long()
        turn = _matrices64(st["cos"][at], st["sin"][at], case["halves"])
        for i, (x, w, dy) in enumerate(((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk")))):
            x, w = x[t:t + step].double(), w.double()
            norm = ((x ** 2).sum(-1, keepdim=True) / D + _EPS).sqrt()
            if dy is None:
                y = w * (x / norm)
                y[..., lo:hi] = torch.matmul(y[..., lo:hi], turn.transpose(1, 2).contiguous())
            else:
                g = dy[t:t + step].double()
                g[..., lo:hi] = torch.matmul(g[..., lo:hi].clone(), turn)  # the transposed rotation
                grads[i] += (g * x / norm).sum((0, 1))
                g = g * w
                # d (x / norm): the projection of g out of x's direction
                y = g / norm - x * (g * x).sum(-1, keepdim=True) / (D * norm ** 3)
            ys[i].append(y)
    out = [torch.cat(y) for y in ys]
    return tuple(out if case["direction"] == "forward" else out + grads)


def _stored64(cache, i, where):
    """Values in 64 bits of the pages `where` of a cache's keys (0) or values (1)."""
    if own:
        cache = (cache.k, cache.v) if cache.k_scales is None else (cache.k, cache.v, cache.k_scales, cache.v_scales)
    if len(cache) == 2:
        return cache[i][where].double()
    words, scales = cache[i][where].long() & 0xFFFFFFFF, cache[2 + i][where]
    nib = torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1)
    e, m = ((nib >> 1) & 3).double(), (nib & 1).double()
    v = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e - 1)) * torch.where(nib >= 8, -1.0, 1.0)
    return (v.reshape(*scales.shape, 32) * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def _nearest64(x):
    """Blocks of 32 as MXFP4 keeps them: multiples of a power of two, the even
    code of two equally near ones."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)[[0, 2, 4, 6, 1, 3, 5, 7]]
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    power = torch.where(top > 0, torch.floor(torch.log2(top)) - 2, -127.0)
    power = torch.where(torch.exp2(power + 2) > top, power - 1, power).clamp_min(-127.0)
    m = b.abs() / torch.exp2(power)
    best, dist = torch.zeros_like(m), torch.full_like(m, float("inf"))
    for g in grid:  # odd codes come last, so that the first of two equal distances is the even one
        d = (m - g).abs()
        best, dist = torch.where(d < dist, g, best), torch.minimum(d, dist)
    return (torch.copysign(best, b) * torch.exp2(power)).reshape(x.shape)


def _append64(st, case):
    whole = [_stored64(st["cache"], i, slice(None)) for i in (0, 1)]
    slots, page = st["slots"].long(), case["page"]
    for t in range(0, case["tokens"], 1024):
        at = st["positions"][t:t + 1024].long()
        k, v = st["k"][t:t + 1024].double(), st["v"][t:t + 1024].double()
        if case["norm"]:
            k = st["weight"].double() * (k / ((k ** 2).sum(-1, keepdim=True) / case["dim"] + _EPS).sqrt())
        if case["rope"]:
            lead = k[..., :case["rope"]]
            turn = _matrices64(st["cos"][at], st["sin"][at], case["halves"])
            k = torch.cat([torch.matmul(lead, turn.transpose(1, 2).contiguous()), k[..., case["rope"]:]], -1)
        for i, x in enumerate((k, v)):
            new = x if case["cache"] == "bf16" else _nearest64(x)
            mine = slots[t:t + 1024]
            whole[i][mine[mine >= 0] // page, :, mine[mine >= 0] % page] = new[mine >= 0]
    return tuple(whole)


def _attend64(st, case):
    H, G, Q = case["kv_heads"], case["heads"] // case["kv_heads"], case["queries"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        where = st["table"][b, :-(-n // case["page"])].long()
        k, v = (_stored64(st["cache"], i, where).transpose(0, 1).flatten(1, 2)[:, :n] for i in (0, 1))
        for lo in range(0, Q, 512):
            hi = min(Q, lo + 512)
            limit = torch.arange(n - Q + lo, n - Q + hi, device="cuda")[:, None]
            key = torch.arange(n, device="cuda")
            hidden = key > limit
            if case["window"]:
                hidden = hidden | (key <= limit - case["window"])
            for h in range(case["heads"]):
                s = st["q"][b * Q + lo:b * Q + hi, h].double() @ k[h // G].t() * st["scale"]
                s = s.masked_fill(hidden, float("-inf"))
                if st["sinks"] is not None:
                    s = torch.cat([s, st["sinks"][h].double().expand(hi - lo, 1)], 1)
                out[b * Q + lo:b * Q + hi, h] = torch.softmax(s, 1)[:, :n] @ v[h // G]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _norm64, "append": _append64, "attend": _attend64}[case["op"]](st, case)
