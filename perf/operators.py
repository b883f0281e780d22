"""The 8-bit linear operators as they are measured: cases, inputs, plain forms and definitions.

The operators serve a decoder block with 8-bit linears (e4m3 values, one fp32 scale
for each block of 128):

* ``norm``: RMSNorm, with or without the residual's addition, quantised rows out;
* ``silu``: SwiGLU of packed [gate | up] rows, quantised rows out;
* ``quantize``: bf16 rows (a scale for each 128 columns of a row) or a weight (a
  scale for each 128 x 128 block) to 8 bits;
* ``linear``: y = x W^T of quantised rows and weight, bf16 out, with or without a
  residual added.

A block of values y has a = max(max|y|, 2^-100), scale a / 448 and q = e4m3(y * (448 / a)).
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-6
BLOCK = 128
TOP = 448.0  # the largest e4m3 value
LOWEST_AMAX = 2.0**-100
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # the norm between two layers of a decode step: 8 candidate rows at the S10 width
        {"name": "norm_decode", "op": "norm", "rows": 8, "hidden": 768, "residual": True, "pad": 0},
        # the first norm of a batched prompt: odd row count, a width that ends inside a block, rows of a wider buffer
        {"name": "norm_ragged", "op": "norm", "rows": 1999, "hidden": 2000, "residual": False, "pad": 48},
        # the norm between two layers of a large batched prompt
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "hidden": 8192, "residual": True, "pad": 0},
        # SwiGLU of a decode step at the S10 width
        {"name": "silu_decode", "op": "silu", "rows": 8, "f": 2048},
        # SwiGLU of a large batched prompt, odd row count
        {"name": "silu_prompt", "op": "silu", "rows": 12001, "f": 10240},
        # the attention output of 512 prompt tokens, before its projection
        {"name": "quantize_rows", "op": "quantize", "rows": 512, "cols": 768, "weight": False, "pad": 0},
        # a weight when a model is loaded
        {"name": "quantize_weight", "op": "quantize", "rows": 16384, "cols": 8192, "weight": True, "pad": 0},
        # qkv projection of a decode step at the S10 widths: latency
        {"name": "linear_decode", "op": "linear", "rows": 8, "n": 1280, "k": 768, "residual": False},
        # one token through a wide down projection, residual added: bound by the weight's bytes
        {"name": "linear_token", "op": "linear", "rows": 1, "n": 8192, "k": 14336, "residual": True},
        # a ragged decode batch
        {"name": "linear_batch", "op": "linear", "rows": 77, "n": 10000, "k": 5008, "residual": False},
        # the gate/up projection of a keystroke batch's prompts at the S10 widths
        {"name": "linear_prefill", "op": "linear", "rows": 500, "n": 4096, "k": 768, "residual": False},
        # a large batched prompt: bound by the tensor cores
        {"name": "linear_prompt", "op": "linear", "rows": 8192, "n": 8192, "k": 8192, "residual": True},
    ]


def _log(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(["norm", "silu", "quantize", "linear", "linear"])
    while True:
        if op == "norm":
            c = {"op": op, "rows": _log(rng, 1, 16384), "hidden": _log(rng, 64, 16384, 16),
                 "residual": rng.random() < 0.6, "pad": rng.choice([0, 0, 16, 80])}
            size, most = c["rows"] * c["hidden"], 16384 * 8192
        elif op == "silu":
            c = {"op": op, "rows": _log(rng, 1, 16384), "f": _log(rng, 64, 16384, 16)}
            size, most = c["rows"] * c["f"], 12001 * 10240
        elif op == "quantize":
            c = {"op": op, "rows": _log(rng, 1, 16384), "cols": _log(rng, 64, 16384, 16),
                 "weight": rng.random() < 0.4, "pad": rng.choice([0, 0, 16, 80])}
            size, most = c["rows"] * c["cols"], 16384 * 8192
        else:
            c = {"op": op, "rows": _log(rng, 1, 8192), "n": _log(rng, 64, 16384, 8), "k": _log(rng, 64, 16384, 16),
                 "residual": rng.random() < 0.4}
            size, most = c["rows"] * c["n"] * c["k"], 8192**3
        if size <= most:
            return c


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    if op == "norm":
        t, h = case["rows"], case["hidden"]
        moved = t * h * ((2 + 2 + 2 + 1) if case["residual"] else (2 + 1)) + 4 * t * _blocks(h) + 2 * h
        return {"bytes": moved, "flops": 6 * t * h}
    if op == "silu":
        t, f = case["rows"], case["f"]
        return {"bytes": t * f * 5 + 4 * t * _blocks(f), "flops": 7 * t * f}
    if op == "quantize":
        t, c = case["rows"], case["cols"]
        scales = _blocks(t) * _blocks(c) if case["weight"] else t * _blocks(c)
        return {"bytes": 3 * t * c + 4 * scales, "flops": 2 * t * c}
    t, n, k = case["rows"], case["n"], case["k"]
    scales = t * _blocks(k) + _blocks(n) * _blocks(k)
    return {"bytes": t * k + n * k + 4 * scales + t * n * (4 if case["residual"] else 2), "flops": 2 * t * n * k}


# ---- inputs ------------------------------------------------------------------
def _activations(gen, rows, cols, width=None):
    """Rows as a decoder has them: channels of unlike size, a few of them large, and every 97th row empty (the
    padding of a batch). `width`: the row length of the buffer that they lie in."""
    width = width or cols
    x = torch.randn((rows, width), generator=gen, device="cuda", dtype=torch.float32)
    x *= torch.exp(0.5 * torch.randn((1, width), generator=gen, device="cuda"))
    x *= 1 + 19 * (torch.rand((1, width), generator=gen, device="cuda") < 0.004)
    x[96::97] = 0
    return x.to(torch.bfloat16)[:, :cols]


def _weight(gen, n, k):
    w = torch.randn((n, k), generator=gen, device="cuda", dtype=torch.float32)
    return (w * 0.02).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "norm":
        t, h = case["rows"], case["hidden"]
        x = _activations(gen, t, h, h + case["pad"])
        g = (1 + 0.1 * torch.randn(h, generator=gen, device="cuda")).to(torch.bfloat16)
        if not case["residual"]:
            return {"case": case, "x": x, "g": g}
        r = _activations(gen, t, h)
        # the next layer's residual stream goes to a buffer of the program's
        return {"case": case, "x": x, "g": g, "r": r, "r_out": torch.empty_like(r)}
    if op == "silu":
        return {"case": case, "x": _activations(gen, case["rows"], 2 * case["f"])}
    if op == "quantize":
        t, c = case["rows"], case["cols"]
        if case["weight"]:
            return {"case": case, "x": _weight(gen, t, c + case["pad"])[:, :c]}
        return {"case": case, "x": _activations(gen, t, c, c + case["pad"])}
    t, n, k = case["rows"], case["n"], case["k"]
    q, s = _quantize(_activations(gen, t, k).float(), 1)
    wq, ws = _quantize(_weight(gen, n, k).float(), BLOCK)
    state = {"case": case, "q": q, "s": s, "wq": wq, "ws": ws}
    if case["residual"]:
        state["r"] = torch.randn((t, n), generator=gen, device="cuda").to(torch.bfloat16)
    return state


# ---- plain forms -------------------------------------------------------------
def _quantize(y, tall):
    """e4m3 values and scales of the fp32 matrix y in blocks of `tall` rows x 128 columns."""
    t, c = y.shape
    tb, cb = -(-t // tall), _blocks(c)
    if tb * tall != t or cb * BLOCK != c:
        y = F.pad(y, (0, cb * BLOCK - c, 0, tb * tall - t))
    y = y.view(tb, tall, cb, BLOCK)
    amax = y.abs().amax(dim=(1, 3)).clamp(min=LOWEST_AMAX)
    q = (y * (TOP / amax)[:, None, :, None]).view(tb * tall, cb * BLOCK)[:t, :c]
    return q.to(E4M3).contiguous(), amax / TOP


def _spread(scale, tall, rows, cols):
    """The scale of each value of a [rows, cols] matrix."""
    s = scale.repeat_interleave(BLOCK, dim=1)[:, :cols]
    return s if tall == 1 else s.repeat_interleave(tall, dim=0)[:rows]


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        s = state["x"].float()
        out = {}
        if case["residual"]:
            s = s + state["r"].float()
            out["residual"] = s.to(torch.bfloat16)
        y = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + EPS) * state["g"].float()
        out["q"], out["scale"] = _quantize(y, 1)
        return out
    if op == "silu":
        g, u = state["x"].float().chunk(2, dim=1)
        q, s = _quantize(g / (1 + torch.exp(-g)) * u, 1)
        return {"q": q, "scale": s}
    if op == "quantize":
        q, s = _quantize(state["x"].float(), BLOCK if case["weight"] else 1)
        return {"q": q, "scale": s}
    t, n, k = case["rows"], case["n"], case["k"]
    x = state["q"].float() * _spread(state["s"], 1, t, k)
    w = state["wq"].float() * _spread(state["ws"], BLOCK, n, k)
    y = x @ w.t()
    if case["residual"]:
        y = state["r"].float() + y
    return {"y": y.to(torch.bfloat16)}


def _framework(state):
    from aios_b200 import _lib
    from aios_b200.kernel import ops

    case = state["case"]
    op = case["op"]
    if op == "norm":
        if not case["residual"]:
            q, s = ops.rmsnorm_fp8(state["x"], state["g"], EPS)
            return {"q": q, "scale": s}
        q, s = ops.fused_add_rmsnorm_fp8(state["x"], state["r"], state["g"], EPS, residual_out=state["r_out"])
        return {"q": q, "scale": s, "residual": state["r_out"]}
    if op == "silu":
        q, s = ops.silu_and_mul_fp8(state["x"])
        return {"q": q, "scale": s}
    if op == "quantize":
        q, s = (ops.quantize_weight_fp8 if case["weight"] else ops.quantize_fp8)(state["x"])
        return {"q": q, "scale": s}
    if case["residual"]:
        y = ops.linear_fp8(state["q"], state["s"], state["wq"], state["ws"], epilogue=_lib.EPI_ADD,
                           residual=state["r"])
    else:
        y = ops.linear_fp8(state["q"], state["s"], state["wq"], state["ws"])
    return {"y": y}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- definitions in 64 bits --------------------------------------------------
def _e4m3(v):
    """The nearest e4m3 value of each v (ties to the even mantissa): 3 mantissa bits, exponents from -6, at most 448."""
    _, e = torch.frexp(v.abs())  # |v| in [2^(e-1), 2^e)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_blocks(y, tall):
    """_quantize's values and scales by a walk over the blocks of columns, in 64 bits."""
    t, c = y.shape
    q = torch.empty_like(y)
    scales = []
    groups = torch.arange(t, device=y.device) // tall
    count = -(-t // tall)
    for at in range(0, c, BLOCK):
        part = y[:, at : at + BLOCK]
        top = torch.zeros(count, dtype=y.dtype, device=y.device).scatter_reduce(
            0, groups, part.abs().max(dim=1).values, "amax")
        scale = torch.clamp(top, min=LOWEST_AMAX) / TOP
        q[:, at : at + BLOCK] = _e4m3(part / scale[groups][:, None])
        scales.append(scale)
    return q, torch.stack(scales, dim=1)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        s = state["x"].double()
        out = {}
        if case["residual"]:
            s = s + state["r"].double()
            out["residual"] = s
        rms = torch.sqrt(torch.linalg.vector_norm(s, dim=1, keepdim=True) ** 2 / case["hidden"] + EPS)
        out["q"], out["scale"] = _exact_blocks(s / rms * state["g"].double(), 1)
        return out
    if op == "silu":
        f = case["f"]
        g, u = state["x"][:, :f].double(), state["x"][:, f:].double()
        q, s = _exact_blocks(torch.sigmoid(g) * g * u, 1)
        return {"q": q, "scale": s}
    if op == "quantize":
        q, s = _exact_blocks(state["x"].double(), BLOCK if case["weight"] else 1)
        return {"q": q, "scale": s}
    t, n, k = case["rows"], case["n"], case["k"]
    y = state["r"].double() if case["residual"] else torch.zeros((t, n), dtype=torch.float64, device="cuda")
    heights = torch.arange(n, device="cuda") // BLOCK
    for b in range(_blocks(k)):  # block by block: an integer-like product, then its two scales
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        p = state["q"][:, at].double() @ state["wq"][:, at].double().t()
        p *= state["s"][:, b, None].double()
        y += p * state["ws"][:, b].double()[heights][None, :]
    return {"y": y}
