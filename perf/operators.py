"""The 8-bit floating-point (e4m3) dense layer of the library and what feeds it, as measured workloads.

Four operators: ``quantize_fp8`` (bf16 to e4m3 with a scale per block: 1 x 128 for activations, 128 x 128 for
weights), ``rms_norm`` (residual addition, root-mean-square norm, bf16 and / or e4m3 result), ``gemm_fp8`` (e4m3
product with the block scales applied, bias and activation) and ``linear_fp8`` (``quantize_fp8`` of bf16 rows and
``gemm_fp8`` in one call).  ``own`` chooses between the plain form, elementary torch operations in 32 bits, and the
library's entry points.

The block rule, for the values x of one block: amax = max |x| (a NaN stays a NaN); scale = amax / 448, or 1 where
amax < 2^-117 (a block of zeros); code = e4m3(x * (448 / amax)), round half to even.  Scales of activations are
stored block-major, [ceil(width / 128), rows]; those of weights [ceil(rows / 128), ceil(width / 128)].
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
TINY = 2.0 ** -117
FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16

# Caps of what draw() makes: the largest listed case of each operator.
MAX_QUANTIZE = 262144 * 1536
MAX_NORM = 262144 * 1024
MAX_GEMM = 262144 * 1536 * 1024
MAX_LINEAR = 65536 * 1024 * 1024


def listed() -> list[dict]:
    return [
        # One position (64 tokens, embedding width 1024): what a search with a single leaf quantises per layer.
        {"name": "quantize_rows_64x1024", "op": "quantize", "rows": 64, "width": 1024, "block_rows": 1},
        # The hidden rows of the feed-forward at the benchmark's batch of 4096 positions.
        {"name": "quantize_rows_262144x1536", "op": "quantize", "rows": 262144, "width": 1536, "block_rows": 1},
        # A large weight matrix at load time, one scale per 128 x 128 block; ragged on both sides.
        {"name": "quantize_weight_8190x8200", "op": "quantize", "rows": 8190, "width": 8200, "block_rows": 128},
        # One token of a decoder: residual addition, norm, e4m3 row for the product that follows.
        {"name": "rms_norm_1x4096", "op": "rms_norm", "rows": 1, "width": 4096, "skip": True, "out": False, "quant": True},
        # A ragged batch of an odd width, bf16 result only.
        {"name": "rms_norm_5003x1111", "op": "rms_norm", "rows": 5003, "width": 1111, "skip": True, "out": True,
         "quant": False},
        # The residual stream at batch 4096: new residual, bf16 row and e4m3 row in one pass.
        {"name": "rms_norm_262144x1024", "op": "rms_norm", "rows": 262144, "width": 1024, "skip": True, "out": True,
         "quant": True},
        # One token through a 4096 x 4096 projection: the weight's bytes are all there is.
        {"name": "gemm_1x4096x4096", "op": "gemm", "m": 1, "n": 4096, "k": 4096, "bias": False, "activation": "none",
         "out": "bf16"},
        # One position through feed-forward dense1.
        {"name": "gemm_64x1536x1024", "op": "gemm", "m": 64, "n": 1536, "k": 1024, "bias": True, "activation": "mish",
         "out": "bf16"},
        # Ragged everywhere: tokens, policy-sized output (1858, rows not 16-byte aligned), inner width 1000; f32 logits.
        {"name": "gemm_777x1858x1000", "op": "gemm", "m": 777, "n": 1858, "k": 1000, "bias": True, "activation": "none",
         "out": "f32"},
        # Feed-forward dense1 with mish at batch 4096: the largest.
        {"name": "gemm_262144x1536x1024", "op": "gemm", "m": 262144, "n": 1536, "k": 1024, "bias": True,
         "activation": "mish", "out": "bf16"},
        # Eight tokens in flight through an output projection, bf16 rows in.
        {"name": "linear_8x8192x2048", "op": "linear", "m": 8, "n": 8192, "k": 2048, "bias": True, "activation": "none"},
        # The attention output projection at batch 1024, bf16 rows in.
        {"name": "linear_65536x1024x1024", "op": "linear", "m": 65536, "n": 1024, "k": 1024, "bias": True,
         "activation": "none"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    op = rng.choice(["quantize", "rms_norm", "gemm", "gemm", "linear"])
    if op == "quantize":
        width = _log_int(rng, 32, 8192)
        return {"op": op, "rows": _log_int(rng, 1, min(262144, MAX_QUANTIZE // width)), "width": width,
                "block_rows": rng.choice([1, 1, BLOCK])}
    if op == "rms_norm":
        width = _log_int(rng, 32, 8192)
        quant = rng.choice([True, True, False])
        return {"op": op, "rows": _log_int(rng, 1, min(262144, MAX_NORM // width)), "width": width,
                "skip": rng.choice([True, True, False]), "out": not quant or rng.choice([True, False]), "quant": quant}
    n, k = _log_int(rng, 16, 8192), _log_int(rng, 64, 8192)
    most = min(262144, (MAX_GEMM if op == "gemm" else MAX_LINEAR) // (n * k), 262144 * 1024 // max(n, k))
    case = {"op": op, "m": _log_int(rng, 1, max(1, most)), "n": n, "k": k, "bias": rng.choice([True, False]),
            "activation": rng.choice(["none", "none", "mish", "relu", "swish"])}
    if op == "gemm":
        case["out"] = rng.choice(["bf16", "bf16", "f32"])
    return case


# ------------------------------------------------------------------ inputs

def _rows(gen, rows: int, width: int) -> torch.Tensor:
    """Activations: channels of different strength, as a residual stream has them."""
    strength = torch.exp(torch.randn(width, generator=gen, device="cuda"))
    return (torch.randn((rows, width), generator=gen, device="cuda") * strength).to(BF16)


def _pitched(rows: int, width: int, dtype: torch.dtype) -> torch.Tensor:
    """An 8-bit matrix whose rows start at multiples of 16 bytes, as a program that feeds TMA keeps it."""
    return torch.zeros((rows, -(-width // 16) * 16), dtype=dtype, device="cuda")[:, :width]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        rows, width, block_rows = case["rows"], case["width"], case["block_rows"]
        x = _rows(gen, rows, width) if block_rows == 1 else (
            torch.randn((rows, width), generator=gen, device="cuda") * 0.02).to(BF16)
        blocks = -(-width // BLOCK)
        shape = (blocks, rows) if block_rows == 1 else (-(-rows // BLOCK), blocks)
        return {"case": case, "x": x, "q": _pitched(rows, width, FP8), "scale": torch.empty(shape, device="cuda")}
    if op == "rms_norm":
        rows, width = case["rows"], case["width"]
        state = {"case": case, "x": torch.randn((rows, width), generator=gen, device="cuda").to(BF16),
                 "skip": _rows(gen, rows, width) if case["skip"] else None,
                 "gamma": (1 + 0.1 * torch.randn(width, generator=gen, device="cuda")).to(BF16)}
        state["residual"] = torch.empty_like(state["x"]) if case["skip"] else None
        state["out"] = torch.empty_like(state["x"]) if case["out"] else None
        state["q"] = _pitched(rows, width, FP8) if case["quant"] else None
        state["scale"] = torch.empty((-(-width // BLOCK), rows), device="cuda") if case["quant"] else None
        return state
    m, n, k = case["m"], case["n"], case["k"]
    a = _rows(gen, m, k)
    w = (torch.randn((n, k), generator=gen, device="cuda") / math.sqrt(k)).to(BF16)
    state = {"case": case, "w": _pitched(n, k, FP8),
             "bias": (0.1 * torch.randn(n, generator=gen, device="cuda")).to(BF16) if case["bias"] else None}
    codes, state["w_scale"] = _quantize(w, BLOCK)
    state["w"].copy_(codes)
    if op == "gemm":
        state["a"] = _pitched(m, k, FP8)
        codes, state["a_scale"] = _quantize(a, 1)
        state["a"].copy_(codes)
        state["out"] = torch.empty((m, n), dtype=BF16 if case["out"] == "bf16" else torch.float32, device="cuda")
    else:
        state["a"] = a
        state["scratch_q"] = torch.empty((m, -(-k // 16) * 16), dtype=FP8, device="cuda")
        state["scratch_scale"] = torch.empty((-(-k // BLOCK), m), device="cuda")
        state["out"] = torch.empty((m, n), dtype=BF16, device="cuda")
    return state


# ------------------------------------------------------------------ plain form

def _quantize(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes [rows, width] and scales of 32-bit or bf16 values."""
    rows, width = x.shape
    blocks, row_blocks = -(-width // BLOCK), -(-rows // block_rows)
    padded = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - width, 0, row_blocks * block_rows - rows))
    tiles = padded.reshape(row_blocks, block_rows, blocks, BLOCK)
    amax = tiles.abs().amax(dim=(1, 3), keepdim=True)
    small = amax < TINY
    top = torch.full_like(amax, E4M3_MAX)  # tensor by tensor: torch divides by a number as it multiplies by its inverse
    scale = torch.where(small, 1.0, amax / top)
    inverse = torch.where(small, 1.0, top / amax)
    codes = (tiles * inverse).clamp(-E4M3_MAX, E4M3_MAX).to(FP8)
    codes = codes.reshape(row_blocks * block_rows, blocks * BLOCK)[:rows, :width]
    scale = scale.reshape(row_blocks, blocks)
    return codes, (scale.t().contiguous() if block_rows == 1 else scale)


def _activate(y: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "mish":
        return y * torch.tanh(torch.clamp(y, min=0) + torch.log1p(torch.exp(-y.abs())))
    if activation == "relu":
        return torch.clamp(y, min=0)
    if activation == "swish":
        return y / (1 + torch.exp(-y))
    return y


def _product(a, a_scale, w, w_scale, bias, activation: str, dtype: torch.dtype) -> torch.Tensor:
    (m, k), n = a.shape, w.shape[0]
    a32 = a.float() * a_scale.t().repeat_interleave(BLOCK, dim=1)[:, :k]
    w32 = w.float() * w_scale.repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    y = a32 @ w32.t()
    if bias is not None:
        y = y + bias.float()
    return _activate(y, activation).to(dtype)


def _rms_norm(s: dict) -> dict:
    v = s["x"].float()
    result = {}
    if s["skip"] is not None:
        v = v + s["skip"].float()
        result["residual"] = v.to(BF16)
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * s["gamma"].float()
    if s["out"] is not None:
        result["out"] = y.to(BF16)
    if s["q"] is not None:
        result["q"], result["scale"] = _quantize(y, 1)
    return result


_ops = None


def _library():
    global _ops
    if _ops is None:
        from lczero_triton_b200 import ops
        _ops = ops
    return _ops


def run(state: dict):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        ops = _library()
        if op == "quantize":
            ops.quantize_fp8(s["q"], s["scale"], s["x"], block_rows=case["block_rows"])
            return {"q": s["q"], "scale": s["scale"]}
        if op == "rms_norm":
            ops.rms_norm(s["out"], s["x"], s["gamma"], epsilon=1e-6, skip=s["skip"], residual_out=s["residual"],
                         q_out=s["q"], q_scale=s["scale"])
            return {name: s[name] for name in ("residual", "out", "q", "scale") if s[name] is not None}
        if op == "gemm":
            return ops.gemm_fp8(s["out"], s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"],
                                activation=case["activation"])
        return ops.linear_fp8(s["out"], s["a"], s["w"], s["w_scale"], s["bias"], s["scratch_q"], s["scratch_scale"],
                              activation=case["activation"])
    if op == "quantize":
        q, scale = _quantize(s["x"], case["block_rows"])
        return {"q": q, "scale": scale}
    if op == "rms_norm":
        return _rms_norm(s)
    if op == "gemm":
        a, a_scale = s["a"], s["a_scale"]
    else:
        a, a_scale = _quantize(s["a"], 1)
    return _product(a, a_scale, s["w"], s["w_scale"], s["bias"], case["activation"], s["out"].dtype)


def work(case: dict) -> dict:
    if case["op"] in ("quantize", "rms_norm"):
        rows, width = case["rows"], case["width"]
        blocks = -(-width // BLOCK)
        if case["op"] == "quantize":
            scales = blocks * (rows if case["block_rows"] == 1 else -(-rows // BLOCK))
            return {"bytes": rows * width * 3 + scales * 4, "flops": rows * width * 3}
        per = 2 + (4 if case["skip"] else 0) + (2 if case["out"] else 0) + (1 if case["quant"] else 0)
        return {"bytes": rows * width * per + width * 2 + (rows * blocks * 4 if case["quant"] else 0),
                "flops": rows * width * 7}
    m, n, k = case["m"], case["n"], case["k"]
    blocks = -(-k // BLOCK)
    moved = n * k + blocks * -(-n // BLOCK) * 4 + (n * 2 if case["bias"] else 0)
    if case["op"] == "gemm":
        moved += m * k + m * blocks * 4 + m * n * (2 if case["out"] == "bf16" else 4)
    else:
        moved += m * k * 2 + m * n * 2
    return {"bytes": moved, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, half to even: four significant bits, exponent -6 at the least."""
    _, exponent = torch.frexp(x)  # |x| in [2^(exponent - 1), 2^exponent)
    step = torch.exp2((exponent - 1).clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_blocks(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and the scale of every element, both [rows, width]."""
    rows, width = x.shape
    whole = x.new_zeros((-(-rows // block_rows) * block_rows, -(-width // BLOCK) * BLOCK))
    whole[:rows, :width] = x
    top = whole.abs().unflatten(1, (-1, BLOCK)).amax(dim=2).unflatten(0, (-1, block_rows)).amax(dim=1)
    scale = torch.where(top < TINY, torch.ones_like(top), top / E4M3_MAX)
    spread = torch.kron(scale, scale.new_ones((block_rows, BLOCK)))[:rows, :width]
    return _exact_e4m3(x / spread), scale


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        q, scale = _exact_blocks(s["x"].double(), case["block_rows"])
        return {"q": q, "scale": scale.t() if case["block_rows"] == 1 else scale}
    if op == "rms_norm":
        v = s["x"].double()
        result = {}
        if s["skip"] is not None:
            v = v + s["skip"].double()
            result["residual"] = v
        y = v * s["gamma"].double() * torch.rsqrt(v.square().sum(dim=1, keepdim=True) / case["width"] + 1e-6)
        if s["out"] is not None:
            result["out"] = y
        if s["q"] is not None:
            result["q"], scale = _exact_blocks(y, 1)
            result["scale"] = scale.t()
        return result
    k = case["k"]
    w = s["w"].double()
    for j in range(0, k, BLOCK):
        w[:, j:j + BLOCK] *= s["w_scale"][:, j // BLOCK].double().repeat_interleave(BLOCK)[:case["n"], None]
    if op == "gemm":
        a, scale = s["a"].double(), s["a_scale"].double().t()
    else:
        a, scale = _exact_blocks(s["a"].double(), 1)
    for j in range(0, k, BLOCK):
        a[:, j:j + BLOCK] *= scale[:, j // BLOCK, None]
    y = torch.einsum("mk,nk->mn", a, w)
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["activation"] == "mish":
        y = torch.nn.functional.mish(y)
    elif case["activation"] == "relu":
        y = torch.relu(y)
    elif case["activation"] == "swish":
        y = torch.nn.functional.silu(y)
    return y
