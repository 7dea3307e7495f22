"""The MXFP4 and routed-expert operators, measured: the calls that a program
makes of them, over the sizes it makes them with.

    listed()            the cases looked at one by one
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what the program holds before the call (on the GPU)
    run(state)          one pass; returns its outputs whole
    work(case)          the bytes and flops a pass cannot do without
    exact(case, seed)   the outputs in 64 bits, from the definitions

Kinds ("op"):
    quantize  a matrix to MXFP4 (blocks of 32 along a row: one power of two
              and 32 e2m1 numbers), and the values that this stands for
    mm        y = x . W^T of T tokens with an MXFP4 weight; x in bf16 or f32,
              or in MXFP4 too
    experts   the same for T tokens of K experts each: rows in expert order,
              each expert's rows times its own matrix
    route     tokens sorted by expert and back: "forward" sorts the ids, lays
              the tokens' rows out in expert order and adds the experts'
              results up with the router's weights; "backward" is the gradient
              of the last two

`own` false: plain torch in 32 bits; true: the library's calls.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # the magnitudes of e2m1


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minirun-app_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import minirun_hip

    return minirun_hip


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the input of one decode step's projection: launches are all of it
        {"name": "quantize_t1_7168", "op": "quantize", "rows": 1, "cols": 7168, "dtype": "bf16"},
        # a checkpoint's f32 matrix made into an MXFP4 weight while it loads
        {"name": "quantize_24576x1536_f32", "op": "quantize", "rows": 24576, "cols": 1536, "dtype": "f32"},
        # the output projection of one decode step, 128 heads: weights from HBM
        {"name": "mm_t1_7168x16384", "op": "mm", "tokens": 1, "out_features": 7168, "in_features": 16384,
         "x": "bf16", "y": "bf16"},
        # a serving batch of 37 decode steps
        {"name": "mm_t37_24576x1536", "op": "mm", "tokens": 37, "out_features": 24576, "in_features": 1536,
         "x": "bf16", "y": "bf16"},
        # a prompt with bf16 activations
        {"name": "mm_t4096_24576x1536", "op": "mm", "tokens": 4096, "out_features": 24576, "in_features": 1536,
         "x": "bf16", "y": "bf16"},
        # a prompt with activations in MXFP4 too
        {"name": "mm_t4096_7168x16384_mxfp4", "op": "mm", "tokens": 4096, "out_features": 7168, "in_features": 16384,
         "x": "mxfp4", "y": "bf16"},
        # routed experts of one decode step: 8 of 128
        {"name": "experts_t1_e128_k8_768x2048", "op": "experts", "tokens": 1, "experts": 128, "per_token": 8,
         "out_features": 768, "in_features": 2048, "x": "bf16", "rows": "tokens"},
        # the experts' second projection for a prompt chunk: rows that the
        # first one left in expert order
        {"name": "experts_t200_e128_k8_2048x768_sorted", "op": "experts", "tokens": 200, "experts": 128, "per_token": 8,
         "out_features": 2048, "in_features": 768, "x": "bf16", "rows": "sorted"},
        # a whole prompt with activations in MXFP4
        {"name": "experts_t4096_e128_k8_768x2048_mxfp4", "op": "experts", "tokens": 4096, "experts": 128, "per_token": 8,
         "out_features": 768, "in_features": 2048, "x": "mxfp4", "rows": "tokens"},
        # one decode step's way to the experts and back
        {"name": "route_t1_e128_k8_7168", "op": "route", "direction": "forward", "tokens": 1, "experts": 128,
         "per_token": 8, "dim": 7168, "dtype": "bf16", "dropped": 0.0},
        # a prompt's, half of the experts on another GPU
        {"name": "route_t4096_e128_k8_7168_half", "op": "route", "direction": "forward", "tokens": 4096, "experts": 128,
         "per_token": 8, "dim": 7168, "dtype": "bf16", "dropped": 0.5},
        # the gradient for an odd number of tokens
        {"name": "route_t2001_e256_k6_2048_backward", "op": "route", "direction": "backward", "tokens": 2001,
         "experts": 256, "per_token": 6, "dim": 2048, "dtype": "bf16", "dropped": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "mm", "mm", "experts", "experts", "route"])
    if op == "quantize":
        cols = 32 * _log(rng, 1, 512)
        return {"op": op, "rows": _log(rng, 1, min(24576, 37_000_000 // cols)), "cols": cols,
                "dtype": rng.choice(["bf16", "f32"])}
    if op == "mm":
        out, inp = _log(rng, 16, 24576), 32 * _log(rng, 1, 512)
        return {"op": op, "tokens": _log(rng, 1, max(1, min(4096, 480_000_000_000 // (out * inp)))), "out_features": out,
                "in_features": inp, "x": rng.choice(["bf16", "bf16", "f32", "mxfp4"] if out * inp < 2e7
                                                    else ["bf16", "bf16", "mxfp4"]),
                "y": rng.choice(["bf16", "f32"])}
    if op == "experts":
        return {"op": op, "tokens": _log(rng, 1, 4096), "experts": rng.choice([8, 60, 128, 256]),
                "per_token": rng.randint(1, 8), "out_features": _log(rng, 128, 2048),
                "in_features": 32 * _log(rng, 4, 64), "x": rng.choice(["bf16", "mxfp4"]),
                "rows": rng.choice(["tokens", "sorted"])}
    dim = _log(rng, 64, 7168)
    return {"op": op, "direction": rng.choice(["forward", "backward"]), "tokens": _log(rng, 1, 4096),
            "experts": rng.choice([8, 60, 128, 256]), "per_token": rng.randint(1, 8),
            "dim": dim if rng.random() < 0.25 else -(-dim // 8) * 8, "dtype": rng.choice(["bf16", "bf16", "f32"]),
            "dropped": rng.choice([0.0, 0.0, 0.3])}


# ---------------------------------------------------------------- plain MXFP4
def _power(byte):
    """2^(byte - 127) in f32; NaN at 255."""
    bits = torch.where(byte == 0, 0x00400000, byte << 23)
    return torch.where(byte == 255, 0x7FC00000, bits).to(torch.int32).view(torch.float32)


def _quantize(x):
    """Codes [rows, cols] (0..15) and scale bytes [rows, cols / 32] of x, int32."""
    b = x.float().reshape(x.shape[0], -1, 32)
    top = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    exponent = top.view(torch.int32) >> 23  # floor(log2 top) + 127; 0 below the normal numbers
    byte = torch.where(finite, (exponent - 2).clamp_min(0), 255)
    up = ((254 - byte).clamp_min(1) << 23).to(torch.int32).view(torch.float32)  # 2^(127 - byte)
    m = (b * up[..., None]).abs()
    code = ((m > 0.25).int() + (m >= 0.75).int() + (m > 1.25).int() + (m >= 1.75).int() + (m > 2.5).int()
            + (m >= 3.5).int() + (m > 5.0).int())
    code = torch.where(finite[..., None], code + 8 * torch.signbit(b).int(), 0)
    return code.reshape(x.shape).to(torch.int32), byte.to(torch.int32)


def _pack(code):
    c = code.reshape(*code.shape[:-1], -1, 8)
    word = c[..., 0].clone()
    for j in range(1, 8):
        word |= c[..., j] << (4 * j)
    return word


def _values(packed, scales):
    """f32 [..., cols] of packed words [..., cols / 8] and bytes [..., cols / 32]."""
    shift = torch.arange(0, 32, 4, device=packed.device, dtype=torch.int32)
    code = (packed[..., None] >> shift) & 15
    table = torch.tensor(_GRID + tuple(-g for g in _GRID), device=packed.device)
    v = table[code.long()].reshape(*scales.shape, 32)
    return (v * _power(scales.int())[..., None]).reshape(*packed.shape[:-1], -1)


# ---------------------------------------------------------------- inputs
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return (std * torch.randn(*shape, generator=self.g, device="cuda")).to(dtype)

    def mxfp4(self, rows, cols, std, lead=()):
        """A matrix (or a stack) of normal values as its quantizer leaves it."""
        n = rows * (lead[0] if lead else 1)
        code, byte = _quantize(self.normal(n, cols, std=std, dtype=torch.float32))
        return (_pack(code).reshape(*lead, rows, cols // 8).contiguous(),
                byte.to(torch.uint8).reshape(*lead, rows, cols // 32).contiguous())

    def ids(self, tokens, experts, per_token):
        """The best `per_token` experts of each token, some liked more than others."""
        logits = torch.randn(tokens, experts, generator=self.g, device="cuda")
        logits += 0.5 * torch.randn(experts, generator=self.g, device="cuda")
        return logits.topk(per_token, dim=1)


def _order(ids, experts):
    """Stable order of the pairs (token, slot) by expert; ids outside [0, experts) have no row."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    pair_of_row = torch.sort(key, stable=True).indices
    counts = torch.zeros(experts + 1, dtype=torch.long, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:experts].cumsum(0)])
    row = torch.empty_like(key)
    row[pair_of_row] = torch.arange(key.numel(), device=ids.device)
    row = torch.where(key < experts, row, -1)
    kept = torch.arange(key.numel(), device=ids.device) < offsets[-1]
    pair_of_row = torch.where(kept, pair_of_row, -1)
    return offsets.int(), pair_of_row.int(), row.reshape(ids.shape).int()


def prepare(case, seed):
    op = case["op"]
    r = _Rand(seed)
    st = {"op": op, "case": dict(case)}
    if op == "quantize":
        # rows of their own size each, and now and then a value far from the others
        x = r.normal(case["rows"], case["cols"], dtype=torch.float32)
        x *= torch.exp(torch.randn(case["rows"], 1, generator=r.g, device="cuda"))
        x *= torch.where(torch.rand(x.shape, generator=r.g, device="cuda") < 0.001, 20.0, 1.0)
        st["x"] = x.to(_DT[case["dtype"]])
        return st
    if op == "route":
        T, E, K, D, dt = case["tokens"], case["experts"], case["per_token"], case["dim"], _DT[case["dtype"]]
        logits, ids = r.ids(T, E, K)
        st["weights"] = torch.softmax(logits, dim=1)
        # experts held elsewhere come first in the numbering: their ids are below zero here
        st["local"] = E - round(E * case["dropped"])
        st["ids"] = (ids - (E - st["local"])).to(torch.int32).contiguous()
        if case["direction"] == "forward":
            st["x"] = r.normal(T, D, dtype=dt)
            st["rows"] = torch.zeros(T * K, D, dtype=dt, device="cuda")  # dispatched rows; those past the last stay zero
        else:
            st["d_out"], st["d_xs"] = r.normal(T, D, dtype=dt), r.normal(T * K, D, dtype=dt)
            st["d_rows"] = torch.zeros(T * K, D, dtype=dt, device="cuda")
            st["order"] = _order(st["ids"], st["local"])
        st["ys"] = r.normal(T * K, D, dtype=dt)
        if own and case["direction"] == "backward":
            st["order"] = _lib().ExpertOrder(*st["order"], experts=st["local"])
        return st
    T, out, inp = case["tokens"], case["out_features"], case["in_features"]
    rows = T
    if op == "experts":
        E, K = case["experts"], case["per_token"]
        ids = r.ids(T, E, K).indices.to(torch.int32).contiguous()
        st["order"] = _order(ids, E)
        rows = T * K if case["rows"] == "sorted" else T
    st["x"] = r.mxfp4(rows, inp, 1.0) if case["x"] == "mxfp4" else r.normal(rows, inp, dtype=_DT[case["x"]])
    st["w"] = r.mxfp4(out, inp, inp ** -0.5, (case["experts"],) if op == "experts" else ())
    if own:
        M = _lib()
        st["w"] = M.MXFP4Weights(*st["w"])
        if case["x"] == "mxfp4":
            st["x"] = M.MXFP4Weights(*st["x"])
        if op == "experts":
            st["order"] = M.ExpertOrder(*st["order"], experts=case["experts"])
    return st


# ---------------------------------------------------------------- one pass
def _run_own(st):
    M = _lib()
    op, case = st["op"], st["case"]
    if op == "quantize":
        return M.mxfp4_dequantize(M.mxfp4_quantize(st["x"]), dtype=st["x"].dtype)
    if op == "mm":
        return M.mxfp4_mm(st["x"], st["w"], out_dtype=_DT[case["y"]])
    if op == "experts":
        return M.mxfp4_expert_mm(st["x"], st["w"], st["order"], sorted_rows=case["rows"] == "sorted",
                                 out_dtype=torch.bfloat16)
    if case["direction"] == "forward":
        order = M.expert_sort(st["ids"], st["local"])
        xs = M.expert_dispatch(st["x"], order, out=st["rows"])
        out = M.expert_combine(st["ys"], order, st["weights"])
        return {"offsets": order.offsets, "pair_of_row": order.pair_of_row, "row_of_pair": order.row_of_pair,
                "xs": xs, "out": out}
    d_rows, d_weights = M.expert_combine_backward(st["d_out"], st["ys"], st["order"], st["weights"], out=st["d_rows"])
    return {"d_rows": d_rows, "d_weights": d_weights, "d_x": M.expert_dispatch_backward(st["d_xs"], st["order"])}


def _run_plain(st):
    op, case = st["op"], st["case"]
    if op == "quantize":
        code, byte = _quantize(st["x"])
        table = torch.tensor(_GRID + tuple(-g for g in _GRID), device=code.device)
        v = table[code.long()].reshape(*byte.shape, 32) * _power(byte)[..., None]
        return v.reshape(st["x"].shape).to(st["x"].dtype)
    if op in ("mm", "experts"):
        x = _values(*st["x"]) if case["x"] == "mxfp4" else st["x"].float()
        if op == "mm":
            return (x @ _values(*st["w"]).t()).to(_DT[case["y"]])
        offsets, pair_of_row, _ = st["order"]
        if case["rows"] == "tokens":
            x = x[pair_of_row.long() // case["per_token"]]
        y = torch.empty(x.shape[0], case["out_features"], dtype=torch.bfloat16, device=x.device)
        ends = offsets.tolist()
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            if hi > lo:
                y[lo:hi] = (x[lo:hi] @ _values(st["w"][0][e], st["w"][1][e]).t()).to(y.dtype)
        return y
    T, K = st["ids"].shape
    if case["direction"] == "forward":
        offsets, pair_of_row, row_of_pair = _order(st["ids"], st["local"])
        kept = (pair_of_row >= 0)[:, None]
        xs = torch.where(kept, st["x"][pair_of_row.long() // K], st["rows"])
        back = st["ys"].float()[row_of_pair.long().clamp_min(0)]
        w = torch.where(row_of_pair >= 0, st["weights"], 0.0)
        out = torch.zeros(T, case["dim"], device=w.device)
        for j in range(K):
            out += torch.where(row_of_pair[:, j, None] >= 0, w[:, j, None] * back[:, j], 0.0)
        return {"offsets": offsets, "pair_of_row": pair_of_row, "row_of_pair": row_of_pair, "xs": xs,
                "out": out.to(st["ys"].dtype)}
    _, pair_of_row, row_of_pair = st["order"]
    at, has = row_of_pair.long().clamp_min(0), row_of_pair >= 0
    pair = pair_of_row.long().clamp_min(0)
    d_out = st["d_out"].float()
    d_rows = d_out[pair // K] * st["weights"].reshape(-1)[pair][:, None]
    d_rows = torch.where((pair_of_row >= 0)[:, None], d_rows.to(st["ys"].dtype), st["d_rows"])
    d_weights = torch.stack([(d_out * st["ys"][at[:, j]].float()).sum(1) for j in range(K)], 1)
    d_x = torch.zeros_like(d_out)
    for j in range(K):
        d_x += torch.where(has[:, j, None], st["d_xs"][at[:, j]].float(), 0.0)
    return {"d_rows": d_rows, "d_weights": torch.where(has, d_weights, 0.0), "d_x": d_x.to(st["d_xs"].dtype)}


def run(st):
    return _run_own(st) if own else _run_plain(st)


# ---------------------------------------------------------------- minimal work
def _mxfp4_bytes(n):
    return n // 2 + n // 32


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["cols"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * size * n, "flops": 2 * n}
    if op == "route":
        T, K, E, D = case["tokens"], case["per_token"], case["experts"], case["dim"]
        size = 2 if case["dtype"] == "bf16" else 4
        pairs = T * K
        rows = pairs * (E - round(E * case["dropped"])) / E  # of which there are, about
        if case["direction"] == "forward":
            # ids and weights; three index arrays; x and the rows out; the results and their sums
            return {"bytes": round(8 * pairs + 8 * pairs + size * D * (T + rows + rows + T)), "flops": round(2 * rows * D)}
        return {"bytes": round(12 * pairs + size * D * (T + 3 * rows + T)), "flops": round(4 * rows * D)}
    T, out, inp = case["tokens"], case["out_features"], case["in_features"]
    x_bytes = {"bf16": lambda n: 2 * n, "f32": lambda n: 4 * n, "mxfp4": _mxfp4_bytes}[case["x"]]
    if op == "mm":
        return {"bytes": x_bytes(T * inp) + _mxfp4_bytes(out * inp) + (2 if case["y"] == "bf16" else 4) * T * out,
                "flops": 2 * T * out * inp}
    E, K = case["experts"], case["per_token"]
    used = E * (1 - (1 - K / E) ** T)  # experts that some token is routed to
    return {"bytes": round(x_bytes((T * K if case["rows"] == "sorted" else T) * inp) + used * _mxfp4_bytes(out * inp)
                           + 4 * T * K + 2 * T * K * out), "flops": 2 * T * K * out * inp}


# ---------------------------------------------------------------- 64 bits
def _values64(w):
    """An MXFP4 operand's values from its words and bytes, in 64 bits: sign,
    2-bit exponent and 1-bit mantissa of each nibble."""
    packed, scales = (w.packed, w.scales) if own and not isinstance(w, tuple) else w
    words = packed.long() & 0xFFFFFFFF
    nib = torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1)
    e, m = ((nib >> 1) & 3).double(), (nib & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e - 1))
    v = torch.where(nib >= 8, -mag, mag).reshape(*scales.shape, 32)
    return (v * torch.exp2(scales.double() - 127)[..., None]).flatten(-2)


def _quantized64(x):
    """The nearest e2m1 multiple of each block's power of two, the even code of
    two equally near ones."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    # odd codes come last, so that the first of two equal distances is the even one
    grid = grid[[0, 2, 4, 6, 1, 3, 5, 7]]
    for lo in range(0, x.shape[0], 512):
        b = x[lo:lo + 512].double().reshape(-1, x.shape[1] // 32, 32)
        top = b.abs().amax(-1, keepdim=True)
        power = torch.where(top > 0, torch.frexp(top).exponent.double() - 1 - 2, -127.0).clamp_min(-127.0)
        m = b.abs() / torch.exp2(power)
        best, dist = torch.zeros_like(m), torch.full_like(m, float("inf"))
        for g in grid:
            d = (m - g).abs()
            better = d < dist
            best, dist = torch.where(better, g, best), torch.where(better, d, dist)
        out[lo:lo + 512] = (torch.copysign(best, b) * torch.exp2(power)).reshape(-1, x.shape[1])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _quantized64(st["x"])
    if op in ("mm", "experts"):
        x = _values64(st["x"]) if case["x"] == "mxfp4" else st["x"].double()
        if op == "mm":
            return x @ _values64(st["w"]).t()
        order = st["order"]
        offsets, pair = (order.offsets, order.pair_of_row) if own else order[:2]
        packed, scales = (st["w"].packed, st["w"].scales) if own else st["w"]
        y = torch.empty(case["tokens"] * case["per_token"], case["out_features"], dtype=torch.float64, device=x.device)
        for e in range(case["experts"]):
            lo, hi = int(offsets[e]), int(offsets[e + 1])
            if hi > lo:
                xe = x[lo:hi] if case["rows"] == "sorted" else x[pair[lo:hi].long() // case["per_token"]]
                y[lo:hi] = xe @ _values64((packed[e], scales[e])).t()
        return y
    T, K, D = case["tokens"], case["per_token"], case["dim"]
    w64 = st["weights"].double()
    if case["direction"] == "forward":
        xs, out = torch.zeros(T * K, D, dtype=torch.float64, device="cuda"), None
        row_of, lists = [[-1] * K for _ in range(T)], [[] for _ in range(st["local"])]
        for p, e in enumerate(st["ids"].reshape(-1).tolist()):
            if 0 <= e < st["local"]:
                lists[e].append(p)
        offsets, pairs = [0], []
        for of_expert in lists:
            for p in of_expert:
                row_of[p // K][p % K] = len(pairs)
                pairs.append(p)
            offsets.append(len(pairs))
        n = len(pairs)
        pair = torch.tensor(pairs, dtype=torch.long, device="cuda")
        xs[:n] = st["x"].double()[pair // K]
        out = torch.zeros(T, D, dtype=torch.float64, device="cuda")
        out.index_add_(0, pair // K, w64.reshape(-1)[pair, None] * st["ys"][:n].double())
        int_ = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        return {"offsets": int_(offsets), "pair_of_row": int_(pairs + [-1] * (T * K - n)),
                "row_of_pair": int_(row_of).reshape(T, K), "xs": xs, "out": out}
    order = st["order"]
    offsets, pair = (order.offsets, order.pair_of_row) if own else order[:2]
    n = int(offsets[-1])
    pair = pair[:n].long()
    g = st["d_out"].double()[pair // K]
    d_rows = torch.zeros(T * K, D, dtype=torch.float64, device="cuda")
    d_rows[:n] = w64.reshape(-1)[pair, None] * g
    d_weights = torch.zeros(T * K, dtype=torch.float64, device="cuda")
    d_weights[pair] = (g * st["ys"][:n].double()).sum(1)
    d_x = torch.zeros(T, D, dtype=torch.float64, device="cuda").index_add_(0, pair // K, st["d_xs"][:n].double())
    return {"d_rows": d_rows, "d_weights": d_weights.reshape(T, K), "d_x": d_x}
