"""Cases, plain forms and exact values of the 4-bit floating-point linear operators.

Operators: quantisation of rows to microscaled 4-bit floats and back ("quantize"), the product of two such
operands ("product"), the linear layer of 16-bit activations over a 4-bit weight ("linear"), the residual's
addition with the RMSNorm after it and an INT8 output ("norm"), and that norm with a 4-bit output in front of the
product, as a layer of a language model runs them ("layer").

`run` computes an operator in elementary torch operations (`own` false) or through the framework's calls (`own`
true); `exact` computes it in 64 bits from the definition.

Two formats of 4-bit values {0, 0.5, 1, 1.5, 2, 3, 4, 6} with a sign (to the nearest, ties to the even code):
  mxfp4  blocks of 32 columns; a block's scale is 2^(floor(log2(its absmax)) - 2), within 2^-127 .. 2^127;
  nvfp4  blocks of 16 columns; a row has a scale r = 2^e, e >= -126 the least with absmax <= 2688 * 2^e, and a
         block the scale e4m3(its absmax / 6 / r) on top of it.
Values above 6 become 6.  An INT8 row has the scale absmax / 127.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
EPS = 1e-5


def listed():
    return [
        # The norm in front of a projection, for one decoded token and for a long prompt.
        dict(name="norm_token", op="norm", rows=1, cols=4096, dtype="bf16"),
        dict(name="norm_prompt", op="norm", rows=8190, cols=4096, dtype="fp16"),
        # A projection's weight as it is laid out when a model is loaded.
        dict(name="quantize_weight", op="quantize", rows=16384, cols=4096, dtype="bf16", format="mxfp4"),
        # Rows of a width that fills neither its last block nor its last group of blocks.
        dict(name="quantize_ragged", op="quantize", rows=3607, cols=1044, dtype="fp16", format="nvfp4"),
        # One decoded token through the three projections of attention, with a bias.
        dict(name="linear_token", op="linear", rows=1, cols=4096, outs=12288, dtype="bf16", format="nvfp4", bias=True),
        # A serving batch of decoded tokens through the second projection of an MLP.
        dict(name="linear_batch", op="linear", rows=48, cols=16384, outs=4096, dtype="bf16", format="mxfp4", bias=False),
        # One short prompt.
        dict(name="linear_prompt", op="linear", rows=333, cols=4096, outs=4096, dtype="fp16", format="mxfp4", bias=True),
        # A latent frame of a 720p video (45 x 80 tokens) through the first projection of an MLP.
        dict(name="linear_frame", op="linear", rows=3600, cols=4096, outs=16384, dtype="bf16", format="nvfp4", bias=True),
        # Operands that fill no tile.
        dict(name="product_ragged", op="product", rows=1111, cols=1056, outs=1003, dtype="fp16", format="nvfp4"),
        # Packed documents through an MLP's second projection.
        dict(name="product_packed", op="product", rows=16384, cols=16384, outs=4096, dtype="bf16", format="mxfp4"),
        # Residual, norm and projection of eight decoded tokens, and of a batch of prompts.
        dict(name="layer_tokens", op="layer", rows=8, cols=4096, outs=4096, dtype="bf16", format="nvfp4"),
        dict(name="layer_prompts", op="layer", rows=8192, cols=4096, outs=12288, dtype="bf16", format="mxfp4"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "quantize", "linear", "linear", "linear", "product", "product", "layer"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op != "norm":
        case["format"] = rng.choice(["mxfp4", "nvfp4"])
    whole = rng.choice([1, 8, 32, 32, 128, 256])  # widths that models have are mostly multiples of something
    case["cols"] = max(whole, _log(rng, 64, 16384) // whole * whole)
    if op in ("norm", "quantize"):
        case["rows"] = _log(rng, 1, min(16384, (1 << 26) // case["cols"]))
        return case
    whole = rng.choice([1, 8, 64, 128, 256])
    case["outs"] = max(whole, _log(rng, 64, 16384) // whole * whole)
    case["rows"] = _log(rng, 1, min(16384, (1 << 40) // (case["cols"] * case["outs"])))
    if op == "linear":
        case["bias"] = rng.choice([True, False])
    return case


def work(case):
    m, k, op = case["rows"], case["cols"], case["op"]
    if op == "norm":  # x, the residual and the sum; codes and scales
        return {"bytes": 6.0 * m * k + 2.0 * k + m * k + 4.0 * m, "flops": 0.0}
    four = 0.5 + 1 / BLOCK[case["format"]]
    if op == "quantize":  # to the codes and back to values
        return {"bytes": m * k * (2 + 2 * four + 2), "flops": 0.0}
    n = case["outs"]
    read = {"linear": 2.0, "product": four, "layer": 6.0}[op]
    return {"bytes": m * k * read + n * k * four + 2.0 * m * n, "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------------------------ inputs

def _activations(rows, cols, dtype, g):
    """Rows of unequal size with a few strong channels, as a transformer's activations have them."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.6 * torch.randn(cols, device="cuda", generator=g))
    x *= torch.exp(0.4 * torch.randn(rows, 1, device="cuda", generator=g))
    strong = torch.randint(0, cols, (max(1, cols // 512),), device="cuda", generator=g)
    x[:, strong] *= 12.0
    return x.to(dtype)


def _weight(rows, cols, dtype, g):
    w = torch.randn(rows, cols, device="cuda", generator=g) / math.sqrt(cols)
    w *= torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))
    return w.to(dtype)


def _h3b():
    if "h3b" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-minimaxh3_b200"))
    import h3b
    return h3b


def _kept(x, fmt):
    """A quantised operand that a program keeps: the framework's, or the values that its codes and scales stand for."""
    return _h3b().quantize_fp4(x, fmt) if own else _values(_plain_fp4(x.float(), fmt), x.shape[1])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dt, m, k, op = DTYPES[case["dtype"]], case["rows"], case["cols"], case["op"]
    s = {"case": case, "x": _activations(m, k, dt, g)}
    if op in ("norm", "layer"):
        s["residual"] = (3 * _activations(m, k, torch.float32, g)).to(dt)
        s["norm"] = (1 + 0.2 * torch.randn(k, device="cuda", generator=g)).to(dt)
        s["sum"] = torch.empty_like(s["residual"])
        s["values"] = torch.empty_like(s["residual"])
    if op in ("linear", "product", "layer"):
        s["weight16"] = _weight(case["outs"], k, dt, g)
        s["bias"] = torch.randn(case["outs"], device="cuda", generator=g) if case.get("bias") else None
        # a weight is laid out once, before the calls that use it, and so are rows that several products take
        s["weight"] = _kept(s["weight16"], case["format"])
        s["rows"] = _kept(s["x"], case["format"]) if op == "product" else None
    return s


# ------------------------------------------------------------------------------------ one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    h3b, case = _h3b(), s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "norm":
        h, (q, scale) = h3b.add_rms_norm_quantize(s["x"], s["residual"], s["norm"], eps=EPS, to="int8", out=s["sum"])
        return h, torch.mul(q, scale, out=s["values"]), scale
    if op == "quantize":
        return h3b.dequantize_fp4(h3b.quantize_fp4(s["x"], case["format"]), dt)
    if op == "linear":
        return h3b.fp4_linear(s["x"], s["weight"], s["bias"])
    if op == "product":
        return h3b.fp4_linear_prequantized(s["rows"], s["weight"], out_dtype=dt)
    h, q = h3b.add_rms_norm_quantize(s["x"], s["residual"], s["norm"], eps=EPS, to=case["format"], out=s["sum"])
    return h, h3b.fp4_linear_prequantized(q, s["weight"], out_dtype=dt)


# ---- plain forms

def _round_e2m1(a):
    """|values| to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code."""
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).clamp_max(6.0)


def _plain_fp4(x, fmt):
    """fp32 rows as (4-bit values with their sign [rows, blocks, block], block scales [rows, blocks], row scales)."""
    m, k = x.shape
    b = BLOCK[fmt]
    x = torch.nn.functional.pad(x, (0, -k % b)).view(m, -1, b)
    top = x.abs().amax(-1)
    if fmt == "mxfp4":
        e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
        scale, r = torch.ldexp(torch.ones_like(top), e), torch.ones(m, 1, device=x.device)
        a = torch.ldexp(x.abs(), -e[..., None])
    else:
        row = top.amax(-1, keepdim=True)
        f = torch.frexp(row)  # row = mantissa * 2^exponent, mantissa from 0.5; 2688 = 0.65625 * 2^12
        e = torch.where(row > 0, f.exponent - 12 + (f.mantissa > 0.65625).int(), 0).clamp_min(-126)
        r = torch.ldexp(torch.ones_like(row), e)
        scale = (torch.ldexp(top, -e) / 6).clamp_max(448).to(torch.float8_e4m3fn).float()
        a = torch.ldexp(x.abs(), -e[..., None]) / torch.where(scale > 0, scale, math.inf)[..., None]
    return torch.copysign(_round_e2m1(a), x), scale, r


def _values(parts, k):
    v, scale, r = parts
    return (v * scale[..., None] * r[..., None]).flatten(1)[:, :k]


def _plain_norm(s):
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = h.float()
    return h, f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()


def _run_plain(s):
    case = s["case"]
    op, dt, k = case["op"], DTYPES[case["dtype"]], case["cols"]
    if op == "norm":
        h, y = _plain_norm(s)
        scale = y.abs().amax(-1, keepdim=True) / 127
        return h, (torch.round(y / scale).clamp(-127, 127) * scale).to(dt), scale
    if op == "quantize":
        return _values(_plain_fp4(s["x"].float(), case["format"]), k).to(dt)
    if op == "layer":
        h, y = _plain_norm(s)
        return h, (_values(_plain_fp4(y, case["format"]), k) @ s["weight"].T).to(dt)
    a = s["rows"] if op == "product" else _values(_plain_fp4(s["x"].float(), case["format"]), k)
    y = a @ s["weight"].T
    return (y if s["bias"] is None else y + s["bias"]).to(dt)


# ------------------------------------------------------------------------------------ from the definition, in 64 bits

CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_e2m1(x, scale):
    """The values nearest to x / scale, by comparison with the borders between neighbours times the scale."""
    code = torch.zeros(x.shape, device=x.device, dtype=torch.int64)
    a = x.abs()
    for i in range(7):
        border = (CODES[i] + CODES[i + 1]) / 2 * scale
        code += (a > border) | ((a == border) & (border > 0) if i % 2 else torch.zeros_like(a, dtype=torch.bool))
    v = torch.tensor(CODES, device=x.device, dtype=torch.float64)[torch.where(scale > 0, code, 0)]
    return torch.where(x < 0, -v, v)


def _exact_fp4(x, fmt):
    out = torch.empty_like(x)
    k, b = x.shape[1], BLOCK[fmt]
    r = 1.0
    if fmt == "nvfp4":
        top = x.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(torch.where(top > 0, top, 2688.0) / 2688.0)) - 1
        for _ in range(3):
            e = e + (top > 2688.0 * torch.exp2(e)).double()
        r = torch.exp2(torch.where(top > 0, e, 0.0).clamp_min(-126))
    for c in range(0, k, b):
        part = x[:, c: c + b]
        top = part.abs().amax(1, keepdim=True)
        if fmt == "mxfp4":
            e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
            e = e - (torch.exp2(e) > top).double() + (torch.exp2(e + 1) <= top).double()
            scale = torch.exp2(torch.where(top > 0, e - 2, -127.0).clamp(-127, 127))
            out[:, c: c + b] = _exact_e2m1(part, scale) * scale
        else:
            t = (top / r / 6).clamp_max(448.0)
            step = torch.exp2(torch.floor(torch.log2(t.clamp_min(2.0 ** -6))) - 3)
            scale = torch.round(t / step) * step
            out[:, c: c + b] = _exact_e2m1(part / r, scale) * scale * r
    return out


def exact(case, seed):
    op, k = case["op"], case["cols"]
    s = prepare(case, seed)
    if op in ("norm", "layer"):
        total = s["x"].double() + s["residual"].double()
        h = total.to(s["x"].dtype).double()  # the norm is that of the sum as it is stored
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / k + EPS) * s["norm"].double()
        if op == "norm":
            scale = y.abs().amax(1, keepdim=True) / 127
            return total, torch.round(y / scale).clamp(-127, 127) * scale, scale
        return total, _exact_fp4(y, case["format"]) @ _exact_fp4(s["weight16"].double(), case["format"]).T
    q = _exact_fp4(s["x"].double(), case["format"])
    if op == "quantize":
        return q
    y = q @ _exact_fp4(s["weight16"].double(), case["format"]).T
    return y if s["bias"] is None else y + s["bias"].double()
