"""Performance cases of the operators on device tensors: 4-bit block floating point, its products, and experts.

  quantize       rows of numbers to 4-bit codes with a scale per block, and back to the values the codes stand for
  linear         y = x W^T + bias with 4-bit weights; x is quantized by the call
  expert_linear  the same for rows that belong to different experts, ragged numbers of rows, 4-bit or 16-bit weights,
                 optionally gated: silu(x Wg^T) * (x Wu^T)
  route          the experts of each token and the order of the (token, expert) pairs by expert
  combine        the weighted sum of each token's expert rows, on top of a residual

4-bit values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even column in the low half.
"block32": a scale per 32 columns, a power of two (byte b stands for 2^(b-127), 255 for NaN).  "block16": a scale per 16
columns, e4m3, times one float for the whole tensor.  Tokens of a batch choose experts unevenly, as trained routers do.
Runs from the repository's root.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_BLOCK = {"block32": 32, "block16": 16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _ops():
    package = os.path.abspath("tim-vx_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import deviceops
    return deviceops


def _quantize(name, rows, k, fmt, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "k": k, "fmt": fmt, "dtype": dtype}


def _linear(name, rows, n, k, fmt, dtype, bias):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "fmt": fmt, "dtype": dtype, "bias": bias}


def _experts(name, tokens, top_k, experts, n, k, fmt, dtype, gated, bias):
    return {"name": name, "op": "expert_linear", "tokens": tokens, "top_k": top_k, "experts": experts, "n": n, "k": k,
            "fmt": fmt, "dtype": dtype, "gated": gated, "bias": bias}


def _route(name, tokens, experts, top_k, dtype, normalize):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "normalize": normalize}


def _combine(name, tokens, top_k, n, dtype, residual):
    return {"name": name, "op": "combine", "tokens": tokens, "top_k": top_k, "n": n, "dtype": dtype, "residual": residual}


def listed():
    return [
        # activations of a few requests between two layers, a width that is no multiple of the block
        _quantize("quantize_8x4011_block32", 8, 4011, "block32", "f32"),
        # the activations of a long prompt, or a layer's weights
        _quantize("quantize_8192x8192_block16", 8192, 8192, "block16", "bf16"),
        # one token through the benchmark's 4096-wide fully-connected layer: latency and weight streaming
        _linear("linear_1x4096_block32", 1, 4096, 4096, "block32", "bf16", False),
        # two dozen requests decoding through the 8192-wide layer
        _linear("linear_24x8192_block16", 24, 8192, 8192, "block16", "bf16", True),
        # a long prompt through the same layer, the benchmark's largest product
        _linear("linear_8192x8192_block32", 8192, 8192, 8192, "block32", "bf16", False),
        # a decode step of sixteen requests through the gated first product of 128 small experts: most are read, each for one row or two
        _experts("experts_16x8of128_gated_block32", 16, 8, 128, 768, 2048, "block32", "bf16", True, False),
        # a prompt through the second product of 64 experts, with biases
        _experts("experts_8192x4of64_block16", 8192, 4, 64, 4096, 1408, "block16", "bf16", False, True),
        # a short prompt through experts kept in 16 bits
        _experts("experts_700x2of32_gated_bf16", 700, 2, 32, 1408, 2048, "none", "bf16", True, False),
        # routing of a decode step
        _route("route_16_8of128", 16, 128, 8, "f32", True),
        # routing of a prompt; ties among 16-bit logits
        _route("route_8192_8of256", 8192, 256, 8, "bf16", False),
        # the end of a decode step's expert layer
        _combine("combine_16_8x2048", 16, 8, 2048, "bf16", True),
        # the end of a prompt's expert layer
        _combine("combine_8192_4x4096", 8192, 4, 4096, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cols(rng, lo, hi, step):
    return max(lo, _log(rng, lo, hi) // step * step)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "expert_linear", "expert_linear", "expert_linear", "route", "combine"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    fmt = rng.choice(["block32", "block16"])
    if op == "quantize":
        k = _log(rng, 32, 16384)
        case = _quantize("", min(_log(rng, 1, 16384), max(1, (1 << 26) // k)), k, fmt, rng.choice(["f32", "bf16", "f16"]))
    elif op == "linear":
        case = _linear("", _log(rng, 1, 8192), _log(rng, 128, 8192), _cols(rng, 128, 8192, 32), fmt, dtype, rng.random() < 0.5)
    elif op == "expert_linear":
        experts = _log(rng, 2, 128)
        top_k = rng.randint(1, min(8, experts))
        n, k = _cols(rng, 256, 4096, 8), _cols(rng, 256, 4096, 32)
        fmt = rng.choice(["block32", "block16", "block32", "block16", "none"])
        gated = rng.random() < 0.5
        while experts > 2 and experts * n * k > 5e8:
            experts //= 2
        case = _experts("", _log(rng, 1, 4096), min(top_k, experts), experts, n, k, fmt, dtype, gated, rng.random() < 0.5)
    elif op == "route":
        experts = _log(rng, 4, 512)
        case = _route("", _log(rng, 1, 8192), experts, rng.randint(1, min(8, experts)), rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5)
    else:
        case = _combine("", _log(rng, 1, 8192), rng.randint(1, 8), _cols(rng, 256, 4096, 8), dtype, rng.random() < 0.5)
    del case["name"]
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(g, rows, k, dtype):
    """Normal numbers with a few columns that are an order of magnitude larger, as hidden states have them."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    big = torch.rand(k, generator=g, device="cuda") < 0.01
    return (x * torch.where(big, 12.0, 1.0)).to(_DT[dtype])


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _round_e2m1(v):
    """v >= 0 to the codes of the nearest e2m1 values, ties to the even code."""
    code = (v > 0.25).to(torch.uint8)
    for border, even_above in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (v >= border) if even_above else (v > border)
    return code


def _power(e):
    """2^e in 64 bits, by the exponent's bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _plain_codes(x, fmt, g):
    """Codes [rows][K] and scales [rows][blocks] (as float32 values, the tensor's scale not included) of x, K a multiple of the block."""
    b = _BLOCK[fmt]
    rows, k = x.shape
    x = x.float().reshape(rows, k // b, b)
    amax = x.abs().amax(dim=2)
    if fmt == "block32":
        _, e = torch.frexp(amax)                      # amax = m 2^e, m in [0.5, 1)
        e = torch.where(amax > 0, e - 3, torch.full_like(e, -127)).clamp(min=-127)
        s = _power(e)
        v = (x.double() / s[..., None]).abs()
    else:
        want = (amax.double() / (6.0 * g.double())).clamp(max=448.0)
        _, e = torch.frexp(want)
        step = _power((e - 4).clamp(min=-9))
        s = torch.round(want / step) * step           # torch.round: ties to even
        full = s * g.double()
        v = torch.where(s[..., None] > 0, (x.double() / full[..., None]).abs(), 0.0)
    code = _round_e2m1(v) | torch.where(torch.signbit(x), 8, 0).to(torch.uint8)
    return code.reshape(rows, k), s.float()


def _plain_values(code, s, fmt, g):
    """float32 values of codes [..., K] with scales [..., K / block]."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=code.device)
    v = table[code.int()].reshape(*s.shape, _BLOCK[fmt]) * s[..., None]
    if fmt == "block16":
        v = v * g
    return v.reshape(code.shape)


def _plain_quantized(x, fmt, g):
    k = x.shape[1]
    pad = -k % _BLOCK[fmt]
    if pad:
        x = torch.cat([x, torch.zeros(x.shape[0], pad, dtype=x.dtype, device=x.device)], dim=1)
    return _plain_values(*_plain_codes(x, fmt, g), fmt, g)[:, :k]


def _unpack(codes):
    return torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)


def _scale_bytes(s, fmt):
    if fmt == "block32":
        _, e = torch.frexp(s)
        return (e + 126).to(torch.uint8)
    _, e = torch.frexp(s)
    normal = s >= 2.0 ** -6
    mant = torch.where(normal, s / _power(e - 1).float() * 8 - 8, s * 512)
    return (mant.to(torch.int32) + torch.where(normal, (e + 6) * 8, 0)).to(torch.uint8)


def _scale_values(b, fmt):
    if fmt == "block32":
        return _power(b.int() - 127).float()
    e, m = (b.int() >> 3), (b.int() & 7).float()
    return torch.where(e > 0, (1 + m / 8) * _power(e - 7).float(), m / 512)


def _plain_weight(w, fmt, g):
    return _plain_values(_unpack(w["codes"]), _scale_values(w["scales"], fmt), fmt, g)


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _weights(g, lead, n, k, fmt, dtype):
    """Weights as a checkpoint has them: 16-bit numbers, or codes [..., n, k / 2], scale bytes [..., n, k / block] and the tensors' scales."""
    if fmt == "none":
        return {"w": (torch.randn(*lead, n, k, generator=g, device="cuda") / math.sqrt(k)).to(_DT[dtype])}
    rows = math.prod(lead) * n
    scale = torch.full((math.prod(lead),), 4.5 / math.sqrt(k) / (6 * 256.0), device="cuda") if fmt == "block16" else None
    codes = torch.empty(rows, k // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(rows, k // _BLOCK[fmt], dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 24) // k)
    for r in range(0, rows, step):
        m = min(step, rows - r)
        c, s = _plain_codes(torch.randn(m, k, generator=g, device="cuda") / math.sqrt(k), fmt, scale[0] if fmt == "block16" else None)
        codes[r:r + m] = c[:, 0::2] | (c[:, 1::2] << 4)
        scales[r:r + m] = _scale_bytes(s, fmt)
    return {"codes": codes.reshape(*lead, n, k // 2), "scales": scales.reshape(*lead, n, -1), "scale": scale}


def _routing(g, case):
    """Uneven choices of experts: offsets of the experts' rows in the order by expert, and the token of each row."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    liking = torch.randn(e, generator=g, device="cuda")
    ids = torch.argsort(torch.randn(t, e, generator=g, device="cuda") + liking, dim=1, descending=True)[:, :k].reshape(-1)
    order = torch.sort(ids, stable=True).indices
    counts = torch.bincount(ids, minlength=e)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), counts.cumsum(0)])
    return offsets.int(), (order // k).int()


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"op": op, "case": case}
    dtype = case["dtype"]
    if op in ("quantize", "linear", "expert_linear"):
        rows = case["tokens"] if op == "expert_linear" else case["rows"]
        s["x"] = _activations(g, rows, case["k"], dtype)
        # a calibrated scale for the activations: the largest block reaches 6 x 448 at 48
        s["x_scale"] = torch.tensor([48.0 / (6 * 448.0)], device="cuda") if case["fmt"] == "block16" else None
    if op == "linear":
        s["weight"] = _weights(g, (), case["n"], case["k"], case["fmt"], dtype)
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
    elif op == "expert_linear":
        n = case["n"] * (2 if case["gated"] else 1)
        s["weight"] = _weights(g, (case["experts"],), n, case["k"], case["fmt"], dtype)
        s["bias"] = torch.randn(case["experts"], n, generator=g, device="cuda") if case["bias"] else None
        s["offsets"], s["row_index"] = _routing(g, case)
    elif op == "route":
        liking = torch.randn(case["experts"], generator=g, device="cuda")
        s["logits"] = (torch.randn(case["tokens"], case["experts"], generator=g, device="cuda") + liking).to(_DT[dtype])
    elif op == "combine":
        t, k, n = case["tokens"], case["top_k"], case["n"]
        s["z"] = torch.randn(t * k, n, generator=g, device="cuda").to(_DT[dtype])
        s["slots"] = torch.randperm(t * k, generator=g, device="cuda").reshape(t, k).int()
        s["weights"] = torch.softmax(torch.randn(t, k, generator=g, device="cuda"), dim=1)
        s["residual"] = torch.randn(t, n, generator=g, device="cuda").to(_DT[dtype]) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if s["op"] == "expert_linear":
        s["bounds"] = s["offsets"].tolist()
    if own:
        ops = _ops()
        s["ops"] = ops
        fmt = case.get("fmt")
        if "weight" in s:
            w = s["weight"]
            s["handle"] = w["w"] if fmt == "none" else ops.Fp4Weight(w["codes"], w["scales"], fmt, w["scale"], gated=case.get("gated", False))
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def _silu(v):
    return v / (1 + torch.exp(-v))


def _run_own(s):
    ops, case, op = s["ops"], s["case"], s["op"]
    if op == "quantize":
        return ops.dequantize_fp4(ops.quantize_fp4(s["x"], case["fmt"], scale=s["x_scale"]), s["x"].dtype)
    if op == "linear":
        return ops.linear(s["x"], s["handle"], bias=s["bias"], x_scale=s["x_scale"])
    if op == "expert_linear":
        return ops.expert_linear(s["x"], s["handle"], s["offsets"], row_index=s["row_index"], bias=s["bias"], gated=case["gated"], x_scale=s["x_scale"])
    if op == "route":
        r = ops.route_experts(s["logits"], case["top_k"], normalize=case["normalize"])
        return r.ids, r.weights, r.offsets, r.row_index, r.slots
    return ops.combine_experts(s["z"], s["slots"], s["weights"], residual=s["residual"])


def run(state):
    if own:
        return _run_own(state)
    s, case, op = state, state["case"], state["op"]
    if op == "quantize":
        return _plain_quantized(s["x"], case["fmt"], s["x_scale"]).to(s["x"].dtype)
    if op == "linear":
        w = _plain_weight(s["weight"], case["fmt"], s["weight"]["scale"])
        y = _plain_quantized(s["x"], case["fmt"], s["x_scale"]) @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return y.to(s["x"].dtype)
    if op == "expert_linear":
        return _plain_experts(s, case)
    if op == "route":
        return _plain_route(s, case)
    y = (s["z"].float()[s["slots"].long()] * s["weights"][..., None]).sum(dim=1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["z"].dtype)


def _plain_experts(s, case):
    fmt, b = case["fmt"], s["bounds"]
    x = s["x"].float() if fmt == "none" else _plain_quantized(s["x"], fmt, s["x_scale"])
    x = x[s["row_index"].long()]
    y = torch.empty(x.shape[0], case["n"], dtype=s["x"].dtype, device=x.device)
    for e in range(case["experts"]):
        if b[e] == b[e + 1]:
            continue
        w = s["weight"]
        if fmt == "none":
            we = w["w"][e].float()
        else:
            we = _plain_weight({"codes": w["codes"][e], "scales": w["scales"][e]}, fmt, None if w["scale"] is None else w["scale"][e])
        h = x[b[e]:b[e + 1]] @ we.t()
        if s["bias"] is not None:
            h = h + s["bias"][e]
        if case["gated"]:
            h = _silu(h[:, :case["n"]]) * h[:, case["n"]:]
        y[b[e]:b[e + 1]] = h.to(y.dtype)
    return y


def _plain_route(s, case):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = s["logits"].float()
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    ids, chosen = top.indices[:, :k], top.values[:, :k]
    p = torch.exp(chosen - top.values[:, :1])
    total = p.sum(1, keepdim=True) if case["normalize"] else torch.exp(logits - top.values[:, :1]).sum(1, keepdim=True)
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * k, device=order.device)
    ends = (flat[:, None] == torch.arange(e, device=flat.device)).sum(0).cumsum(0)
    offsets = torch.cat([torch.zeros(1, dtype=ends.dtype, device=ends.device), ends])
    return ids.int(), p / total, offsets.int(), (order // k).int(), slots.reshape(t, k).int()


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case):
    op, size = case["op"], _SIZE[case["dtype"]]
    if op == "quantize":
        return {"bytes": 2 * case["rows"] * case["k"] * size, "flops": 0}
    if op in ("linear", "expert_linear"):
        n, k, fmt = case["n"], case["k"], case["fmt"]
        wn = n * (2 if case.get("gated") else 1)
        per = wn * k * size if fmt == "none" else wn * k // 2 + wn * k // _BLOCK[fmt]
        if op == "linear":
            x, rows, read = case["rows"], case["rows"], 1
        else:
            x, rows = case["tokens"], case["tokens"] * case["top_k"]
            # experts that at least one row goes to, were the choices even
            read = case["experts"] * (1 - (1 - case["top_k"] / case["experts"]) ** case["tokens"])
        return {"bytes": int(read * per) + x * k * size + rows * n * size + (int(read * wn * 4) if case["bias"] else 0), "flops": 2 * rows * wn * k}
    t, k = case["tokens"], case["top_k"]
    if op == "route":
        return {"bytes": t * case["experts"] * size + 16 * t * k + 4 * case["experts"] + 4, "flops": 0}
    return {"bytes": t * k * (case["n"] * size + 8) + t * case["n"] * size * (2 if case["residual"] else 1), "flops": 2 * t * k * case["n"]}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------

def _powers():
    return torch.tensor([2.0 ** i for i in range(-149, 128)], dtype=torch.float64, device="cuda")


def _e4m3_table():
    v = [m / 512 for m in range(8)] + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64, device="cuda")   # 0 .. 448, in the order of their bytes


def _nearest(table, v):
    """Index of the nearest entry of a rising table, ties to the even index, the ends for what lies outside."""
    hi = torch.searchsorted(table, v.contiguous()).clamp(max=table.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    d_lo, d_hi = v - table[lo], table[hi] - v
    return torch.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)


def _exact_quantized(x, fmt, g):
    b = _BLOCK[fmt]
    rows, k = x.shape
    full = torch.zeros(rows, (k + b - 1) // b * b, dtype=torch.float64, device="cuda")
    full[:, :k] = x.double()
    blocks = full.view(rows, -1, b)
    top = blocks.abs().max(dim=2, keepdim=True).values
    if fmt == "block32":
        powers = _powers()
        below = torch.searchsorted(powers, top.contiguous(), right=True) - 1   # the highest power of two that is not above
        unit = powers[(below - 2).clamp(min=149 - 127)]
    else:
        t = _e4m3_table()
        unit = t[_nearest(t, top / (6 * g.double()))] * g.double()
    grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    mag = torch.where(unit > 0, blocks.abs() / torch.where(unit > 0, unit, 1.0), 0.0)
    return (torch.sign(blocks) * grid[_nearest(grid, mag)] * unit).view(rows, -1)[:, :k]


def _exact_weight(codes, scales, fmt, g):
    grid = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    signed = torch.cat([grid, -grid])
    v = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
    v[:, 0::2], v[:, 1::2] = signed[(codes & 15).long()], signed[(codes >> 4).long()]
    unit = _powers()[scales.long() + 149 - 127] if fmt == "block32" else _e4m3_table()[scales.long()] * g.double()
    return v * unit.repeat_interleave(_BLOCK[fmt], dim=1)


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantized(s["x"], case["fmt"], s["x_scale"])
    if op == "linear":
        w = s["weight"]
        y = torch.matmul(_exact_quantized(s["x"], case["fmt"], s["x_scale"]), _exact_weight(w["codes"], w["scales"], case["fmt"], w["scale"]).T)
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "expert_linear":
        w, fmt, n = s["weight"], case["fmt"], case["n"]
        out = torch.zeros(case["tokens"] * case["top_k"], n, dtype=torch.float64, device="cuda")
        x = s["x"].double() if fmt == "none" else _exact_quantized(s["x"], fmt, s["x_scale"])
        ends = s["offsets"].cpu().numpy()
        for e in np.flatnonzero(np.diff(ends)):
            rows = s["row_index"][ends[e]:ends[e + 1]].long()
            we = w["w"][e].double() if fmt == "none" else _exact_weight(w["codes"][e], w["scales"][e], fmt, None if w["scale"] is None else w["scale"][e])
            h = torch.matmul(x[rows], we.T) + (0 if s["bias"] is None else s["bias"][e].double())
            out[ends[e]:ends[e + 1]] = h[:, :n] * torch.sigmoid(h[:, :n]) * h[:, n:] if case["gated"] else h
        return out
    if op == "route":
        z = s["logits"].double().cpu().numpy()
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        ids = np.argsort(-z, axis=1, kind="stable")[:, :k]
        p = np.exp(z - z.max(axis=1, keepdims=True))
        mine = np.take_along_axis(p, ids, axis=1)
        mine = mine / (mine if case["normalize"] else p).sum(axis=1, keepdims=True)
        pairs = ids.reshape(-1)
        order = np.lexsort((np.arange(t * k), pairs))
        slots = np.argsort(order, kind="stable")
        offsets = np.searchsorted(pairs[order], np.arange(e + 1))
        return (ids.astype(np.int32), mine, offsets.astype(np.int32), (order // k).astype(np.int32), slots.reshape(t, k).astype(np.int32))
    y = torch.einsum("tk,tkn->tn", s["weights"].double(), s["z"].double()[s["slots"].long()])
    return y if s["residual"] is None else y + s["residual"].double()
