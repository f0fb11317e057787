"""Oracle for the e4m3 operators.  TEST INFRASTRUCTURE ONLY.

PARITY UNPINNED: the reference has no 8-bit path, so the rules here are this project's own specification.  Codes and
scales are reproduced bit for bit (the rule is a handful of IEEE fp32 operations); products and norms are evaluated in
64 bits from the codes, scales and bf16 values that the kernels read.
"""

from __future__ import annotations

import torch

BLOCK = 128
TINY = 2.0 ** -117


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of an fp32 / fp64 tensor, half to even, saturated to +-448; NaN stays."""
    x = x.double()
    magnitude = x.abs().clamp(min=2.0 ** -40)
    exponent = torch.floor(torch.log2(magnitude))
    exponent = exponent + (torch.exp2(exponent + 1) <= magnitude).double()  # log2 may round across a power of two,
    exponent = exponent - (torch.exp2(exponent) > magnitude).double()  # either way
    step = torch.exp2(exponent.clamp(min=-6.0) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def quantize(x: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (as fp64 values) [rows, width] and fp32 scales, [blocks, rows] or [row blocks, blocks], of fp32 values."""
    x = x.float()
    rows, width = x.shape
    blocks, row_blocks = -(-width // BLOCK), -(-rows // block_rows)
    padded = x.new_zeros((row_blocks * block_rows, blocks * BLOCK))
    padded[:rows, :width] = x
    tiles = padded.view(row_blocks, block_rows, blocks, BLOCK)
    amax = tiles.abs().amax(dim=(1, 3), keepdim=True)
    zeros = amax < TINY
    top = torch.full_like(amax, 448.0)  # (tensor / number is a multiplication by the inverse in torch)
    scale = torch.where(zeros, torch.ones_like(amax), amax / top)
    inverse = torch.where(zeros, torch.ones_like(amax), top / amax)
    codes = round_e4m3(tiles * inverse).view(row_blocks * block_rows, blocks * BLOCK)[:rows, :width]
    scale = scale.view(row_blocks, blocks)
    return codes, scale.t().contiguous() if block_rows == 1 else scale


def dequantize_rows(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp64 values of codes [rows, width] with block-major scales [blocks, rows]."""
    return codes.double() * scale.double().t().repeat_interleave(BLOCK, dim=1)[:, :codes.shape[1]]


def dequantize_tiles(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    return codes.double() * scale.double().repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]


def activate(y: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "mish":
        return y * torch.tanh(torch.nn.functional.softplus(y))
    if activation == "relu":
        return y.clamp(min=0)
    if activation == "swish":
        return y * torch.sigmoid(y)
    return y


def gemm(a, a_scale, w, w_scale, bias=None, activation: str = "none") -> tuple[torch.Tensor, torch.Tensor]:
    """The product in fp64 and, for the tolerance, sum |a| |w| of the same scaled operands (plus |bias|)."""
    x, v = dequantize_rows(a, a_scale), dequantize_tiles(w, w_scale)
    y, size = x @ v.t(), x.abs() @ v.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return activate(y, activation), size


def rms_norm(x, gamma, epsilon: float, skip=None) -> torch.Tensor:
    v = x.double() if skip is None else x.double() + skip.double()
    return v / torch.sqrt(v.square().mean(dim=1, keepdim=True) + epsilon) * gamma.double()
