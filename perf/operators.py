"""What is measured of the layer operators that feed the decode tail.

Four operators, each through the public entry points of ``lal_b200`` when
``own`` is set and in elementary torch operations when it is not:

* ``norm``   -- residual addition, RMSNorm, output in 8 bits with a scale per
  row (``lal_b200.add_rms_norm_q8``);
* ``swiglu`` -- silu(gate) * up, output in 8 bits with a scale per row
  (``lal_b200.swiglu_q8``);
* ``weights`` -- rows of weights to 4 bits with a scale (and, on demand, a
  minimum) per group of columns, and back (``lal_b200.Q4Weights.quantize`` and
  ``.dequantize``);
* ``matvec`` -- the product of 8-bit vectors with such weights
  (``lal_b200.Q4Weights.matvec``).

An 8-bit row holds q = rint(127 v / max|v|), ties to even, and max|v| / 127.
4-bit weights lie in blocks of 32 columns, 16 bytes each: byte j holds column
j in its low half and column j + 16 in its high half.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"
FLT_MAX = 3.4028234663852886e38

#: the vocabulary and the hidden size of the benchmark's default workload, and
#: the width of that model's feed-forward layer
VOCAB, EMBD, FFN = 152064, 3584, 18944


def listed():
    return [
        # the norm before a layer's products, one stream: nothing but latency
        {"name": "norm_1", "op": "norm", "rows": 1, "n": EMBD, "type": "bf16", "residual": True, "pad": 0},
        # an odd width in rows that are not aligned, no residual (the first norm of a model)
        {"name": "norm_33_odd", "op": "norm", "rows": 33, "n": 769, "type": "f16", "residual": False, "pad": 3},
        # a long prompt
        {"name": "norm_4096", "op": "norm", "rows": 4096, "n": EMBD, "type": "bf16", "residual": True, "pad": 0},
        # the feed-forward activation of one stream, gate and up side by side in one row
        {"name": "swiglu_1", "op": "swiglu", "rows": 1, "n": FFN, "type": "bf16", "pad": 0},
        # the same of a prompt's chunk
        {"name": "swiglu_512", "op": "swiglu", "rows": 512, "n": FFN, "type": "bf16", "pad": 0},
        # a feed-forward matrix quantized at load
        {"name": "weights_ffn", "op": "weights", "rows": FFN, "cols": EMBD, "group": 128, "min": False, "type": "f32"},
        # a small matrix of odd sizes
        {"name": "weights_odd", "op": "weights", "rows": 1001, "cols": 777, "group": 32, "min": True, "type": "bf16"},
        # one stream, the smallest of a layer's products: latency
        {"name": "matvec_1", "op": "matvec", "streams": 1, "rows": EMBD, "cols": EMBD, "group": 32, "min": False, "type": "f32", "pad": 0},
        # a few streams, a matrix of odd sizes, vectors that are not aligned
        {"name": "matvec_5_odd", "op": "matvec", "streams": 5, "rows": 5001, "cols": 1003, "group": 64, "min": True, "type": "f16", "pad": 5},
        # eight streams through the second matrix of the feed-forward layer
        {"name": "matvec_8", "op": "matvec", "streams": 8, "rows": EMBD, "cols": FFN, "group": 32, "min": True, "type": "f32", "pad": 0},
        # sixty-four streams through the first (gate and up in one matrix)
        {"name": "matvec_64", "op": "matvec", "streams": 64, "rows": 2 * FFN, "cols": EMBD, "group": 128, "min": False, "type": "bf16", "pad": 0},
        # a 4-bit LM head for sixteen streams: the largest
        {"name": "matvec_16_head", "op": "matvec", "streams": 16, "rows": VOCAB, "cols": EMBD, "group": 128, "min": False, "type": "f32", "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "weights", "matvec", "matvec"])
    kind = rng.choice(sorted(TYPES))
    pad = rng.choice([0, 0, 3, 8])
    while True:
        if op == "norm":
            c = {"op": op, "rows": _log(rng, 1, 4096), "n": _log(rng, 64, 16384), "type": kind,
                 "residual": rng.random() < 0.7, "pad": pad}
            if c["rows"] * c["n"] <= 2048 * EMBD:
                return c
        elif op == "swiglu":
            c = {"op": op, "rows": _log(rng, 1, 512), "n": _log(rng, 64, FFN), "type": kind, "pad": pad}
            if c["rows"] * c["n"] <= 256 * FFN:
                return c
        elif op == "weights":
            c = {"op": op, "rows": _log(rng, 16, VOCAB), "cols": _log(rng, 64, FFN),
                 "group": rng.choice([32, 64, 128]), "min": rng.random() < 0.5, "type": kind}
            if c["rows"] * c["cols"] <= FFN * EMBD:
                return c
        else:
            c = {"op": op, "streams": _log(rng, 1, 64), "rows": _log(rng, 64, VOCAB), "cols": _log(rng, 64, FFN),
                 "group": rng.choice([32, 64, 128]), "min": rng.random() < 0.5, "type": kind, "pad": pad}
            if c["rows"] * c["cols"] * c["streams"] <= 16 * VOCAB * EMBD and c["rows"] * c["cols"] <= VOCAB * EMBD:
                return c


# ---- inputs ----------------------------------------------------------------------------

def _hidden(g, rows, n, kind, pad):
    """Activations: a standard normal with one value in 200 sixteen times as
    large, in rows `pad` values apart."""
    v = torch.randn(rows, n + pad, generator=g, device=DEV)
    big = torch.rand(rows, n + pad, generator=g, device=DEV) < 0.005
    return torch.where(big, v * 16.0, v).to(TYPES[kind])[:, :n]


def _q4_bytes(cols):
    return (cols + 31) // 32 * 16


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = dict(case)
    op = case["op"]
    if own:
        import lal_b200
        s["lal"] = lal_b200
        s["stream"] = torch.cuda.current_stream().cuda_stream
        s["code"] = {"f32": lal_b200.LAL_TAIL_F32, "bf16": lal_b200.LAL_TAIL_BF16,
                     "f16": lal_b200.LAL_TAIL_F16}[case["type"]]
    if op == "norm":
        rows, n = case["rows"], case["n"]
        s["x"] = _hidden(g, rows, n, case["type"], case["pad"])
        s["r"] = _hidden(g, rows, n, case["type"], case["pad"]) if case["residual"] else None
        s["w"] = 1.0 + 0.2 * torch.randn(n, generator=g, device=DEV)
        s["eps"] = 1e-6
        s["h"] = torch.empty(rows, n, dtype=TYPES[case["type"]], device=DEV) if case["residual"] else None
    elif op == "swiglu":
        rows, n = case["rows"], case["n"]
        both = _hidden(g, rows, 2 * n, case["type"], case["pad"])
        s["gate"], s["up"] = both[:, :n], both[:, n:]
    if op in ("norm", "swiglu"):
        s["q"] = torch.empty(rows, n, dtype=torch.int8, device=DEV)
        s["scale"] = torch.empty(rows, 1, dtype=torch.float32, device=DEV)
        s["y"] = torch.empty(rows, n, dtype=torch.float32, device=DEV)
        return s
    rows, cols, group = case["rows"], case["cols"], case["group"]
    groups = -(-cols // group)
    if op == "weights":
        s["w"] = (0.015 * torch.randn(rows, cols, generator=g, device=DEV)).to(TYPES[case["type"]])
        s["back"] = torch.empty(rows, cols, dtype=torch.float32, device=DEV)
        s["q4"] = torch.empty(rows, _q4_bytes(cols), dtype=torch.uint8, device=DEV)
        s["s4"] = torch.empty(rows, groups, dtype=torch.float16, device=DEV)
        s["m4"] = torch.empty(rows, groups, dtype=torch.float16, device=DEV) if case["min"] else None
    else:
        b = case["streams"]
        # weights that were normal before they were quantized, a few rows at a time
        s["q4"] = torch.empty(rows, _q4_bytes(cols), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 26) // _q4_bytes(cols))
        for r in range(0, rows, step):
            part = s["q4"][r:r + step]
            lo = (torch.randn(part.shape, generator=g, device=DEV) * 2.6 + 8.0).round_().clamp_(1, 15).to(torch.uint8)
            hi = (torch.randn(part.shape, generator=g, device=DEV) * 2.6 + 8.0).round_().clamp_(1, 15).to(torch.uint8)
            part.copy_(lo | (hi << 4))
        size = 0.0055 * (1.0 + 0.2 * torch.randn(rows, groups, generator=g, device=DEV).clamp_(-3, 3))
        s["s4"] = size.half()
        s["m4"] = None
        if case["min"]:
            s["m4"] = (size * (-8.0 + 0.5 * torch.randn(rows, groups, generator=g, device=DEV))).half()
        x = _hidden(g, b, cols, "f32", 0)
        top = x.abs().amax(1, keepdim=True)
        s["xq"] = torch.zeros(b, cols + case["pad"], dtype=torch.int8, device=DEV)[:, :cols]
        s["xq"].copy_((x * (127.0 / top)).round())
        s["sx"] = (top[:, 0] / 127.0).contiguous()
        s["out"] = torch.empty(b, rows, dtype=TYPES[case["type"]], device=DEV)
    if own:
        s["weights"] = s["lal"].Q4Weights(s["q4"].data_ptr(), s["s4"].data_ptr(),
                                          s["m4"].data_ptr() if s["m4"] is not None else None, rows, cols, group)
    return s


# ---- one pass --------------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _own_norm(s):
    x, r, h = s["x"], s["r"], s["h"]
    s["lal"].add_rms_norm_q8(x.data_ptr(), r.data_ptr() if r is not None else None, h.data_ptr() if h is not None else None,
                             s["w"].data_ptr(), s["eps"], s["rows"], s["n"], s["q"].data_ptr(), s["scale"].data_ptr(),
                             s["code"], x_stride=x.stride(0), residual_stride=r.stride(0) if r is not None else None,
                             stream=s["stream"])
    torch.mul(s["q"], s["scale"], out=s["y"])  # the values that the 8 bits stand for
    return {"h": h, "y": s["y"]} if h is not None else {"y": s["y"]}


def _own_swiglu(s):
    gate, up = s["gate"], s["up"]
    s["lal"].swiglu_q8(gate.data_ptr(), up.data_ptr(), s["rows"], s["n"], s["q"].data_ptr(), s["scale"].data_ptr(),
                       s["code"], gate_stride=gate.stride(0), up_stride=up.stride(0), stream=s["stream"])
    torch.mul(s["q"], s["scale"], out=s["y"])
    return {"y": s["y"]}


def _own_weights(s):
    s["weights"].quantize(s["w"].data_ptr(), s["code"], stream=s["stream"])
    s["weights"].dequantize(s["back"].data_ptr(), s["lal"].LAL_TAIL_F32, stream=s["stream"])
    return {"w": s["back"]}


def _own_matvec(s):
    xq = s["xq"]
    s["weights"].matvec(xq.data_ptr(), s["sx"].data_ptr(), s["streams"], s["out"].data_ptr(), s["code"],
                        xq_stride=xq.stride(0), stream=s["stream"])
    return {"y": s["out"]}


_own = {"norm": _own_norm, "swiglu": _own_swiglu, "weights": _own_weights, "matvec": _own_matvec}


def _rows_to_8_bits(v, factor):
    """The values that the 8-bit rows of v * factor stand for; v in 64 bits,
    for the sake of the values next to a border between two steps."""
    top = v.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(v * 127.0 / top), torch.zeros_like(v))
    size = top * factor
    fine = size <= FLT_MAX
    q = torch.where(fine, q, torch.zeros_like(q))
    size = torch.where(fine, size / 127.0, torch.full_like(size, math.nan))
    return q.float() * size.float()


def _plain_norm(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    h = h.to(TYPES[s["type"]])
    v = h.double()
    factor = torch.rsqrt((v * v).mean(1, keepdim=True) + s["eps"])
    y = _rows_to_8_bits(v * s["w"].double(), factor)
    return {"h": h, "y": y} if s["r"] is not None else {"y": y}


def _plain_swiglu(s):
    g, u = s["gate"].double(), s["up"].double()
    return {"y": _rows_to_8_bits(g / (1.0 + torch.exp(-g)) * u, 1.0)}


def _half_up(v):
    """v (64 bits, not negative) in 16 bits, rounded up."""
    h = v.half()
    bits = h.view(torch.int16) + (h.double() < v).to(torch.int16)
    return bits.view(torch.float16)


def _plain_weights(s):
    w, group = s["w"], s["group"]
    out = torch.empty(s["rows"], s["cols"], dtype=torch.float32, device=w.device)
    groups = -(-s["cols"] // group)
    step = max(1, (1 << 24) // s["cols"])
    for r in range(0, s["rows"], step):
        part = w[r:r + step]
        # the last group's missing columns repeat the last one: no extreme is added
        v = torch.cat([part, part[:, -1:].expand(-1, groups * group - s["cols"])], 1).double()
        v = v.view(part.shape[0], groups, group)
        if s["min"]:
            low = v.amin(2, keepdim=True)
            low = -torch.where(low < 0, _half_up((-low).clamp_min(0)).double(), -_half_down(low.clamp_min(0)))
            size = _half_up((v.amax(2, keepdim=True) - low) / 15.0)
            q = torch.where(size > 0, torch.round((v - low) / size.double()), torch.zeros_like(v)).clamp(0, 15)
            back = size.float() * q.float() + low.float()
        else:
            size = _half_up(v.abs().amax(2, keepdim=True) / 7.0)
            q = torch.where(size > 0, torch.round(v / size.double()), torch.zeros_like(v)).clamp(-7, 7)
            back = size.float() * q.float()
        out[r:r + step] = back.view(part.shape[0], -1)[:, :s["cols"]]
    return {"w": out}


def _half_down(v):
    """v (64 bits, not negative) in 16 bits, rounded down, as 64 bits."""
    h = v.half()
    return (h.view(torch.int16) - (h.double() > v).to(torch.int16)).view(torch.float16).double()


def _unpacked(q4, cols):
    """[rows, cols] of the 4-bit numbers."""
    b = q4.view(q4.shape[0], -1, 16)
    return torch.cat([b & 15, b >> 4], 2).view(q4.shape[0], -1)[:, :cols]


def _plain_matvec(s):
    rows, cols, group = s["rows"], s["cols"], s["group"]
    x = s["xq"].float() * s["sx"][:, None]
    y = torch.empty(s["streams"], rows, device=x.device)
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):
        q = _unpacked(s["q4"][r:r + step], cols).float()
        size = s["s4"][r:r + step].float().repeat_interleave(group, 1)[:, :cols]
        if s["min"]:
            w = q * size + s["m4"][r:r + step].float().repeat_interleave(group, 1)[:, :cols]
        else:
            w = (q - 8.0) * size
        y[:, r:r + step] = x @ w.t()
    return {"y": y.to(TYPES[s["type"]])}


_plain = {"norm": _plain_norm, "swiglu": _plain_swiglu, "weights": _plain_weights, "matvec": _plain_matvec}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    op, size = case["op"], 4 if case["type"] == "f32" else 2
    if op == "norm":
        k = case["rows"] * case["n"]
        # x (and the residual and their sum), the weights; 8 bits and the values they stand for
        return {"bytes": k * (size * (3 if case["residual"] else 1) + 1 + 4) + 4 * case["n"] + 4 * case["rows"], "flops": 6 * k}
    if op == "swiglu":
        k = case["rows"] * case["n"]
        return {"bytes": k * (2 * size + 1 + 4) + 4 * case["rows"], "flops": 8 * k}
    rows, cols = case["rows"], case["cols"]
    q4 = rows * (_q4_bytes(cols) + -(-cols // case["group"]) * (4 if case["min"] else 2))
    if op == "weights":
        return {"bytes": rows * cols * (size + 4) + q4, "flops": 6 * rows * cols}
    b = case["streams"]
    return {"bytes": q4 + b * (cols + 4) + b * rows * size, "flops": 2 * b * rows * cols}


# ---- the definition in 64 bits ---------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "swiglu"):
        if op == "norm":
            total = s["x"].to(torch.float64)
            if s["r"] is not None:
                total = (total + s["r"]).to(s["x"].dtype).to(torch.float64)
            v = total * s["w"].to(torch.float64)
            v = v / torch.sqrt(total.square().sum(1, keepdim=True) / case["n"] + s["eps"])
        else:
            g = s["gate"].to(torch.float64)
            v = g * torch.sigmoid(g) * s["up"].to(torch.float64)
        top = v.abs().max(1, keepdim=True).values
        y = torch.round(127.0 * v / top) * (top / 127.0)
        return {"h": total, "y": y} if op == "norm" and case["residual"] else {"y": y}
    rows, cols, group = case["rows"], case["cols"], case["group"]
    of = torch.arange(cols, device=DEV) // group  # the group of each column
    if op == "weights":
        return {"w": torch.cat([_exact_weights(s["w"][r:r + 1024].to(torch.float64), case, of) for r in range(0, rows, 1024)])}
    y = torch.empty(case["streams"], rows, dtype=torch.float64, device=DEV)
    x = s["xq"].to(torch.float64)
    at = torch.arange(cols, device=DEV)
    byte, high = at // 32 * 16 + at % 16, at % 32 >= 16
    step = max(1, (1 << 25) // cols)
    for r in range(0, rows, step):
        raw = s["q4"][r:r + step][:, byte]
        q = torch.where(high, raw >> 4, raw & 15).to(torch.float64)
        size = s["s4"][r:r + step].to(torch.float64)[:, of]
        w = size * q + s["m4"][r:r + step].to(torch.float64)[:, of] if case["min"] else size * (q - 8)
        y[:, r:r + step] = (w @ x.t()).t()
    return {"y": y * s["sx"].to(torch.float64)[:, None]}


def _to_half(v, up):
    """The next 16-bit number at or above (up) or at or below v, as 64 bits."""
    h = v.to(torch.float16)
    wrong = (h.to(torch.float64) < v) if up else (h.to(torch.float64) > v)
    toward = torch.full_like(v, math.inf if up else -math.inf)
    # one step of a 16-bit number: 2^(exponent - 10), 2^-24 at the least
    e = torch.frexp(h.to(torch.float64))[1] - 1
    below = h.to(torch.float64).abs() == torch.exp2(e.to(torch.float64))  # a power of two, towards zero: half the step
    shrink = (h.to(torch.float64) * toward) < 0
    unit = torch.exp2(torch.clamp(e - 10 - (below & shrink).to(e.dtype), min=-24).to(torch.float64))
    return torch.where(wrong, h.to(torch.float64) + (unit if up else -unit), h.to(torch.float64))


def _exact_weights(w, case, of):
    groups = int(of[-1]) + 1
    at = of.expand_as(w)
    high = torch.full((w.shape[0], groups), -math.inf, dtype=w.dtype, device=w.device).scatter_reduce(1, at, w, "amax")
    low = torch.full((w.shape[0], groups), math.inf, dtype=w.dtype, device=w.device).scatter_reduce(1, at, w, "amin")
    if case["min"]:
        low = _to_half(low, False)
        unit = _to_half((high - low) / 15.0, True)
        return torch.round((w - low[:, of]) / unit[:, of]) * unit[:, of] + low[:, of]
    unit = _to_half(torch.maximum(high, -low) / 7.0, True)
    return torch.round(w / unit[:, of]) * unit[:, of]
