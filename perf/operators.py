"""What is measured of the FP8 operators with one scale per block of 128: cases, inputs, plain forms and exact values.

``listed()`` and ``draw(rng)`` give cases, ``prepare(case, seed)`` the inputs on the GPU, ``run(state)`` one pass -- in
elementary torch operations while ``own`` is false, through the library's entry points while it is true -- and
``exact(case, seed)`` the same outputs in 64 bits.  ``work(case)`` counts the bytes and operations a pass cannot do
without.

The operators, for T tokens (E4M3 codes, FP32 scales stored block-major, [ceil(columns / 128), T]):
  residual_norm  residual = bf16(left + right); y = centred RMSNorm(residual); codes and scales of y
  silu_mul       y = silu(gate) * up; codes and scales of y
  quantize       codes and scales of a bf16 tensor
  gemm           bf16(sum over blocks b of sa[b, t] * sw[n / 128, b] * sum over k in b of a[t, k] * w[n, k])
"""
import importlib
import math

import torch

own = False

EPS = 1e-6
BLOCK = 128
TOP = 448.0          # largest E4M3 value
TINY = 2.0 ** -126   # smallest scale of a block that is not all zero


def listed():
    return [
        # one decode step of one request: the norm in front of a projection, latency only
        {"name": "residual_norm 1 token", "op": "residual_norm", "tokens": 1, "cols": 5120, "normalized": False},
        # the ragged end of a prompt, with the bf16 rows that the narrow gate projections of a GDN layer also read
        {"name": "residual_norm 777 tokens", "op": "residual_norm", "tokens": 777, "cols": 5120, "normalized": True},
        # the model's longest prefill panel
        {"name": "residual_norm 8192 tokens", "op": "residual_norm", "tokens": 8192, "cols": 5120, "normalized": False},
        # decode: SwiGLU of the two halves of one merged gate | up row
        {"name": "silu_mul 1 token", "op": "silu_mul", "tokens": 1, "cols": 17408, "merged": True},
        # the longest panel, gate and up from two products
        {"name": "silu_mul 8192 tokens", "op": "silu_mul", "tokens": 8192, "cols": 17408, "merged": False},
        # a short odd tile in front of the attention output projection
        {"name": "quantize 333 tokens", "op": "quantize", "tokens": 333, "cols": 6144},
        # the same at the longest panel
        {"name": "quantize 8192 tokens", "op": "quantize", "tokens": 8192, "cols": 6144},
        # decode of one request: merged gate | up projection, bound by reading the weights
        {"name": "gemm 1 x 34816 x 5120", "op": "gemm", "tokens": 1, "n": 34816, "k": 5120},
        # a decode batch through the MLP down projection: few output rows, a long sum
        {"name": "gemm 48 x 5120 x 17408", "op": "gemm", "tokens": 48, "n": 5120, "k": 17408},
        # one prefill chunk through the GDN qkv projection
        {"name": "gemm 512 x 10240 x 5120", "op": "gemm", "tokens": 512, "n": 10240, "k": 5120},
        # a prompt of odd length through the attention output projection
        {"name": "gemm 1337 x 5120 x 6144", "op": "gemm", "tokens": 1337, "n": 5120, "k": 6144},
        # the longest panel through the merged gate | up projection: the largest call of the model
        {"name": "gemm 8192 x 34816 x 5120", "op": "gemm", "tokens": 8192, "n": 34816, "k": 5120},
    ]


def _log_uniform(rng, low, high, step=1):
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng):
    """One more case of the same ranges: 1 to 8192 tokens, widths on both sides of whole blocks."""
    op = rng.choice(["residual_norm", "silu_mul", "quantize", "gemm", "gemm"])
    tokens = _log_uniform(rng, 1, 8192)
    if op == "residual_norm":
        return {"op": op, "tokens": tokens, "cols": _log_uniform(rng, 256, 8192, 16), "normalized": rng.random() < 0.3}
    if op == "silu_mul":
        return {"op": op, "tokens": tokens, "cols": _log_uniform(rng, 512, 17408, 16), "merged": rng.random() < 0.5}
    if op == "quantize":
        return {"op": op, "tokens": tokens, "cols": _log_uniform(rng, 128, 17408, 16)}
    while True:
        case = {"op": op, "tokens": tokens, "n": _log_uniform(rng, 128, 34816, 8), "k": _log_uniform(rng, 128, 17408, 16)}
        if case["n"] * case["k"] <= 34816 * 5120:  # no more work than the largest listed case
            return case


# ---------------------------------------------------------------------------------------------------- inputs


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _quantize(y):
    """FP32 [rows, cols] -> (E4M3 codes, FP32 scales [blocks, rows]): the plain form of the block quantiser."""
    rows, cols = y.shape
    padded = torch.nn.functional.pad(y, (0, _blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)
    size = padded.abs()
    amax = torch.where(torch.isfinite(size), size, torch.zeros_like(size)).amax(dim=2)
    scale = torch.where(amax == 0, torch.ones_like(amax), torch.clamp(amax / TOP, min=TINY))
    codes = torch.clamp(padded * (1.0 / scale)[:, :, None], -TOP, TOP).to(torch.float8_e4m3fn)
    return codes.view(rows, -1)[:, :cols].contiguous(), scale.t().contiguous()


def _quantize_weight(w):
    """FP32 [n, k] -> (E4M3 codes, FP32 scales [ceil(n / 128), ceil(k / 128)])."""
    n, k = w.shape
    padded = torch.nn.functional.pad(w, (0, _blocks(k) * BLOCK - k, 0, _blocks(n) * BLOCK - n))
    tiles = padded.view(_blocks(n), BLOCK, _blocks(k), BLOCK)
    scale = torch.clamp(tiles.abs().amax(dim=(1, 3)) / TOP, min=TINY)
    codes = (tiles / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(padded.shape)
    return codes[:n, :k].contiguous(), scale.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tokens, op = case["tokens"], case["op"]

    def normal(rows, cols, std=1.0):
        return torch.randn((rows, cols), generator=gen, device="cuda") * std

    def outliers(cols):  # a residual stream has a few channels far above the others
        wide = torch.rand(cols, generator=gen, device="cuda") < 0.01
        return torch.where(wide, 20.0, 1.0)

    state = {"op": op, "tokens": tokens}
    if op == "gemm":
        n, k = case["n"], case["k"]
        codes, scales = _quantize(normal(tokens, k) * outliers(k))
        w_codes, w_scales = _quantize_weight(normal(n, k, 0.02))
        state.update(n=n, k=k, codes=codes, scales=scales, w_codes=w_codes, w_scales=w_scales,
                     out=torch.empty((tokens, n), device="cuda", dtype=torch.bfloat16))
        return state
    cols = case["cols"]
    state.update(cols=cols, codes=torch.empty((tokens, cols), device="cuda", dtype=torch.float8_e4m3fn),
                 scales=torch.empty((_blocks(cols), tokens), device="cuda", dtype=torch.float32))
    if op == "residual_norm":
        state.update(left=(normal(tokens, cols, 2.0) * outliers(cols)).bfloat16(), right=normal(tokens, cols).bfloat16(),
                     weight=normal(1, cols, 0.1).view(-1).bfloat16(),
                     residual=torch.empty((tokens, cols), device="cuda", dtype=torch.bfloat16),
                     normalized=torch.empty((tokens, cols), device="cuda", dtype=torch.bfloat16) if case["normalized"] else None)
    elif op == "silu_mul":
        both = normal(tokens, 2 * cols, 1.5).bfloat16()
        gate, up = both[:, :cols], both[:, cols:]
        state.update(gate=gate if case["merged"] else gate.contiguous(), up=up if case["merged"] else up.contiguous())
    else:
        state.update(x=(normal(tokens, cols) * outliers(cols)).bfloat16())
    return state


# ---------------------------------------------------------------------------------------------------- one pass


def _run_plain(s):
    op = s["op"]
    if op == "gemm":
        n, k = s["n"], s["k"]
        a = s["codes"].float() * s["scales"].t().repeat_interleave(BLOCK, dim=1)[:, :k]
        w = s["w_codes"].float() * s["w_scales"].repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
        return {"out": (a @ w.t()).bfloat16()}
    if op == "residual_norm":
        residual = (s["left"].float() + s["right"].float()).bfloat16()
        r = residual.float()
        y = r * torch.rsqrt(r.square().mean(dim=1, keepdim=True) + EPS) * (1.0 + s["weight"].float())
        codes, scales = _quantize(y)
        got = {"residual": residual, "codes": codes, "scales": scales}
        if s["normalized"] is not None:
            got["normalized"] = y.bfloat16()
        return got
    if op == "silu_mul":
        g = s["gate"].float()
        codes, scales = _quantize(g / (1.0 + torch.exp(-g)) * s["up"].float())
    else:
        codes, scales = _quantize(s["x"].float())
    return {"codes": codes, "scales": scales}


def _run_own(s):
    capi = importlib.import_module("qwen3x-orin_b200").capi
    stream = torch.cuda.current_stream().cuda_stream
    op, tokens = s["op"], s["tokens"]
    if op == "gemm":
        capi.check("q3x_b200_fp8_block_gemm_bf16", s["w_codes"], s["w_scales"], s["codes"], s["scales"], tokens, s["n"], s["k"],
                   s["out"], stream)
        return {"out": s["out"]}
    if op == "residual_norm":
        capi.check("q3x_b200_residual_add_rms_norm_fp8_block", s["left"], s["right"], s["weight"], tokens, s["cols"], EPS,
                   s["residual"], s["normalized"], s["codes"], s["scales"], stream)
        got = {"residual": s["residual"], "codes": s["codes"], "scales": s["scales"]}
        if s["normalized"] is not None:
            got["normalized"] = s["normalized"]
        return got
    if op == "silu_mul":
        capi.check("q3x_b200_silu_mul_fp8_block", s["gate"], s["up"], s["gate"].stride(0), tokens, s["cols"], s["codes"],
                   s["scales"], stream)
    else:
        capi.check("q3x_b200_fp8_block_quantize", s["x"], tokens, s["cols"], s["codes"], s["scales"], stream)
    return {"codes": s["codes"], "scales": s["scales"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- exact values


def _exact_quantized(y):
    """64-bit [rows, cols] -> the values the codes stand for before their rounding, and the scales [blocks, rows]."""
    values, scales = torch.empty_like(y), []
    for first in range(0, y.shape[1], BLOCK):
        part = y[:, first:first + BLOCK]
        top = part.abs().max(dim=1).values / TOP
        top = torch.where(top == 0, torch.ones_like(top), torch.clamp(top, min=TINY))
        values[:, first:first + BLOCK] = part / top[:, None]
        scales.append(top)
    return {"codes": values, "scales": torch.stack(scales)}


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "gemm":
        out = torch.zeros((s["tokens"], s["n"]), device="cuda", dtype=torch.float64)
        for b in range(_blocks(s["k"])):
            a = s["codes"][:, b * BLOCK:(b + 1) * BLOCK].double()
            w = s["w_codes"][:, b * BLOCK:(b + 1) * BLOCK].double()
            a *= s["scales"][b].double()[:, None]
            w *= s["w_scales"][:, b].double().repeat_interleave(BLOCK)[:s["n"], None]
            out.addmm_(a, w.t())
        return {"out": out}
    if op == "residual_norm":
        total = s["left"].double() + s["right"].double()
        r = total.bfloat16().double()  # the norm is that of the rounded residual
        y = r / torch.sqrt((r * r).mean(dim=1, keepdim=True) + EPS) * (s["weight"].double() + 1.0)
        got = {"residual": total, **_exact_quantized(y)}
        if s["normalized"] is not None:
            got["normalized"] = y
        return got
    if op == "silu_mul":
        return _exact_quantized(s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double())
    return _exact_quantized(s["x"].double())


def work(case):
    tokens = case["tokens"]
    if case["op"] == "gemm":
        n, k = case["n"], case["k"]
        scales = 4 * (_blocks(k) * tokens + _blocks(n) * _blocks(k))
        return {"bytes": n * k + tokens * k + scales + 2 * tokens * n, "flops": 2 * tokens * n * k}
    cols = case["cols"]
    result = cols * tokens + 4 * _blocks(cols) * tokens
    if case["op"] == "residual_norm":
        moved = (8 if case["normalized"] else 6) * cols * tokens + 2 * cols
        return {"bytes": moved + result, "flops": 10 * cols * tokens}
    if case["op"] == "silu_mul":
        return {"bytes": 4 * cols * tokens + result, "flops": 10 * cols * tokens}
    return {"bytes": 2 * cols * tokens + result, "flops": 3 * cols * tokens}
