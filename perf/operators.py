"""The 8-bit activation operators of the framework and how they are measured.

Three operators: norm_quantize (residual addition, RMSNorm and rounding to
8-bit codes with a scale a row; without norm and residual it is quantize_rows),
swiglu_quantize (SwiGLU and the same rounding) and linear_int8 (the product of
8-bit rows and 8-bit weights with a scale for each token and channel).

run() computes a case in its plain form, or, with `own` true, through the
framework.  Codes are returned as the values that they stand for, in bf16: two
correct evaluations may round a value on the border of two codes to either.
"""
import importlib
import math

import torch

own = False

PACKAGE = "cl-inference_b200"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
FLT_MIN = 2.0 ** -126
EPS = 1e-5


def _norm(name, m, k, x, residual, norm=True):
    return {"name": name, "op": "norm", "m": m, "k": k, "x": x, "residual": residual, "norm": norm}


def _swiglu(name, m, k, x):
    return {"name": name, "op": "swiglu", "m": m, "k": k, "x": x}


def _linear(name, m, n, k, out, residual=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "out": out, "residual": residual}


def listed():
    return [
        # one decoded token's row ahead of the q/k/v projections: launch latency
        _norm("norm_decode", 1, 4096, "f32", "f32"),
        # a prompt of an 8B model, projections in bf16 and the residual stream in f32
        _norm("norm_prompt", 2048, 4096, "bf16", "f32"),
        # a ragged batch, a width off every vector size, the first layer's norm (no residual yet)
        _norm("norm_ragged", 777, 5001, "f16", "none"),
        # attention output of a 70B model's prompt ahead of the output projection: rounding alone
        _norm("rows_prompt", 1024, 8192, "f32", "none", False),
        # eight decoded tokens ahead of the down projection
        _swiglu("swiglu_decode", 8, 14336, "f32"),
        # a prompt ahead of the down projection
        _swiglu("swiglu_prompt", 2048, 14336, "bf16"),
        # one decoded token through the output projection, onto the residual stream
        _linear("linear_decode", 1, 4096, 4096, "f32", True),
        # sixteen decoded tokens through the gate projection
        _linear("linear_batch", 16, 14336, 4096, "f32"),
        # a ragged batch over an odd weight
        _linear("linear_ragged", 45, 5003, 2051, "f32"),
        # a chunk of a prompt, q/k/v in one weight
        _linear("linear_chunk", 256, 6144, 4096, "f16"),
        # a prompt through an 8B model's gate projection
        _linear("linear_prompt", 2048, 14336, 4096, "bf16"),
        # a long prompt through a 70B model's gate projection
        _linear("linear_long", 4096, 28672, 8192, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number over LOW..HIGH, even over its logarithm; half of them rounded to a multiple of 64 where that fits."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["norm", "swiglu", "linear", "linear"])
    if op == "linear":
        m, n, k = _spread(rng, 1, 4096), _spread(rng, 64, 28672), _spread(rng, 64, 14336)
        out = rng.choice(["f32", "bf16", "f16"])
        most = 4096 * 28672 * 8192
        m = max(1, min(m, most // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "out": out, "residual": out == "f32" and rng.random() < 0.5}
    m, k, x = _spread(rng, 1, 4096), _spread(rng, 64, 28672), rng.choice(["f32", "bf16", "f16"])
    m = max(1, min(m, 2048 * 14336 // k))
    if op == "swiglu":
        return {"op": op, "m": m, "k": k, "x": x}
    norm = rng.random() < 0.75
    return {"op": op, "m": m, "k": k, "x": x, "residual": rng.choice(["none", "f32", x]) if norm else "none", "norm": norm}


def _activations(gen, m, k, scale=1.0):
    """Rows as a decoder's: a normal bulk, each row with its own size, and a few channels many times larger."""
    x = torch.randn((m, k), device="cuda", generator=gen)
    x *= torch.rand((m, 1), device="cuda", generator=gen) + 0.5
    big = torch.rand(k, device="cuda", generator=gen) < 0.002
    return x.mul_(torch.where(big, 8.0 * scale, scale))


def _codes(gen, rows, k):
    """8-bit codes of normal rows, the largest of each row 127, and the rows' scales."""
    c = torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :k]
    for at in range(0, rows, 4096):  # a part of the rows at a time: the f32 values are large
        part = torch.randn((min(4096, rows - at), k), device="cuda", generator=gen)
        c[at:at + 4096] = (part * (127 / part.abs().amax(1, keepdim=True))).round()
    return c, (torch.rand(rows, device="cuda", generator=gen) + 0.5) / 1000


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, k, s = case["m"], case["k"], dict(case)
    if case["op"] == "linear":
        s["xc"], s["xs"] = _codes(gen, m, k)
        s["wc"], s["ws"] = _codes(gen, case["n"], k)
        s["r"] = torch.randn((m, case["n"]), device="cuda", generator=gen) if case["residual"] else None
        return s
    dtype = TYPES[case["x"]]
    if case["op"] == "swiglu":  # gate and up come out of one product, side by side
        both = torch.cat([_activations(gen, m, k, 2.0), _activations(gen, m, k)], 1).to(dtype)
        s["gate"], s["up"] = both[:, :k], both[:, k:]
        return s
    s["t"] = _activations(gen, m, k).to(dtype)
    s["g"] = torch.rand(k, device="cuda", generator=gen) + 0.5 if case["norm"] else None
    s["r"] = _activations(gen, m, k, 2.0).to(TYPES[case["residual"]]) if case["residual"] != "none" else None
    return s


def _round_rows(v, s, fine):
    """Codes of the rows V with scale S times their step, as bf16 values, and the scales."""
    peak = v.abs().amax(1, keepdim=True)
    step = torch.clamp(peak / 127, min=FLT_MIN)
    code = torch.clamp(torch.round(v * (1 / step)), -127, 127)
    scale = torch.where(peak > 0, step * s, torch.ones_like(step))
    fine = fine & torch.isfinite(peak)
    code, scale = torch.where(fine, code, 0.0), torch.where(fine, scale, float("nan"))
    return (code * scale).to(torch.bfloat16), scale[:, 0]


def run(s):
    if own:
        clq = importlib.import_module(PACKAGE)
        if s["op"] == "linear":
            x, w = clq.Int8Rows(s["xc"], s["xs"]), clq.Int8Rows(s["wc"], s["ws"])
            return clq.linear_int8(x, w, dtype=TYPES[s["out"]], residual=s["r"])
        if s["op"] == "swiglu":
            q = clq.swiglu_quantize(s["gate"], s["up"])
            return {"values": q.dequantize(torch.bfloat16), "scales": q.scales}
        if not s["norm"]:
            q = clq.quantize_rows(s["t"])
            return {"values": q.dequantize(torch.bfloat16), "scales": q.scales}
        if s["r"] is None:
            q = clq.norm_quantize(s["t"], s["g"], EPS)
            return {"values": q.dequantize(torch.bfloat16), "scales": q.scales}
        q, total = clq.norm_quantize(s["t"], s["g"], EPS, residual=s["r"])
        return {"values": q.dequantize(torch.bfloat16), "scales": q.scales, "residual": total}
    if s["op"] == "linear":
        y = torch.matmul(s["xc"].float(), s["wc"].float().t()) * s["ws"] * s["xs"][:, None]
        return (y if s["r"] is None else y + s["r"]).to(TYPES[s["out"]])
    if s["op"] == "swiglu":
        gate = s["gate"].float()
        v = gate / (1 + torch.exp(-gate)) * s["up"].float()
        values, scales = _round_rows(v, 1.0, torch.isfinite(v).all(1, keepdim=True))
        return {"values": values, "scales": scales}
    h = s["t"].float() if s["r"] is None else s["t"].float() + s["r"].float()
    if not s["norm"]:
        values, scales = _round_rows(h, 1.0, torch.isfinite(h).all(1, keepdim=True))
        return {"values": values, "scales": scales}
    mean = (h * h).mean(1, keepdim=True)
    values, scales = _round_rows(h * s["g"], 1 / torch.sqrt(mean + EPS), torch.isfinite(mean))
    out = {"values": values, "scales": scales}
    return out if s["r"] is None else {**out, "residual": h.to(s["r"].dtype)}


def work(case):
    m, k = case["m"], case["k"]
    if case["op"] == "linear":
        n = case["n"]
        moved = m * k + n * k + 4 * (m + n) + m * n * (BYTES[case["out"]] + (4 if case["residual"] else 0))
        return {"bytes": moved, "flops": 2 * m * n * k}
    out = 2 * m * k + 4 * m
    if case["op"] == "swiglu":
        return {"bytes": 2 * m * k * BYTES[case["x"]] + out, "flops": 8 * m * k}
    extra = 2 * m * k * BYTES[case["residual"]] if case["residual"] != "none" else 0
    return {"bytes": m * k * BYTES[case["x"]] + extra + out + (4 * k if case["norm"] else 0), "flops": 7 * m * k}


def exact(case, seed):
    """The definition in 64 bits: value = code * scale, code = the nearest whole number to v * 127 / peak."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        parts = []  # the weight's rows a part at a time: they are 64-bit here
        x = s["xc"].double()
        for at in range(0, case["n"], 4096):
            w = s["wc"][at:at + 4096].double() * s["ws"][at:at + 4096, None].double()
            parts.append((x @ w.mT) * s["xs"].double().unsqueeze(1))
        y = torch.cat(parts, 1)
        return y if s["r"] is None else y.add_(s["r"])
    if case["op"] == "swiglu":
        gate = s["gate"].double()
        v, s_row = gate * torch.sigmoid(gate) * s["up"].double(), 1.0
    else:
        v, s_row = s["t"].double(), 1.0
        if s["r"] is not None:
            v = v + s["r"].double()
    out = {}
    if case["op"] == "norm" and s["r"] is not None:
        out["residual"] = v
    if case["op"] == "norm" and case["norm"]:
        s_row = (v.square().mean(1) + EPS).rsqrt()
        v = v * s["g"].double()
    peak = v.abs().amax(1)
    unit = peak / 127 * s_row
    out["values"] = torch.round(v * (127 / peak).unsqueeze(1)) * unit.unsqueeze(1)
    out["scales"] = unit
    return out
