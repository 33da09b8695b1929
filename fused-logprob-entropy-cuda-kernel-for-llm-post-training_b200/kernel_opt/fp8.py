"""Matrix products in 8 bits (e4m3) with a scale for each block of 128.

A weight [O, H] has one fp32 scale per block of 128 x 128 (`quantize_fp8_blocks`, done once);
activations [..., H] one per row and 128 columns (`quantize_fp8_rows`, or straight from the
norm: `fused_residual_rmsnorm_fp8`).  `fp8_linear` multiplies them on the tensor cores, each
block of 128 summed in fp32 and scaled in fp32 registers, the result rounded once.  Inference
only.  No counterpart in the reference.
"""
from __future__ import annotations

import torch

from kernel_opt import _C


def quantize_fp8_rows(x: torch.Tensor):
    """(q, scales) of x [..., H] (bf16 / fp16 / fp32, H at most 16384): q float8_e4m3fn like x,
    scales fp32 [..., ceil(H / 128)]; x is about q * scale."""
    return _C.quantize_fp8_rows(x)


def quantize_fp8_blocks(weight: torch.Tensor):
    """(q, scales) of a weight [O, H]: q float8_e4m3fn [O, H], scales fp32
    [ceil(O / 128), ceil(H / 128)]."""
    return _C.quantize_fp8_blocks(weight)


def fp8_linear(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor,
               weight_scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               activation: str | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """act((x * x_scales) @ (weight * weight_scales).T + bias) + residual: [..., O] in `out_dtype`
    (bf16 / fp16 / fp32), in fp32 up to one rounding.

    x: float8_e4m3fn [..., H]; x_scales: fp32 [..., ceil(H / 128)]; weight: float8_e4m3fn
    [O, H]; weight_scales: fp32 [ceil(O / 128), ceil(H / 128)].  H must be a multiple of 16, at
    most 32768.  `out`: a tensor to write ([N, O], unit stride along O) instead of a new one, whose
    dtype then counts.

    bias: [O] of the output's dtype or fp32; activation: None, 'relu', 'silu', 'gelu' (the erf form) or
    'gelu_tanh'; residual: [..., O] of the output's dtype.  A residual may be `out` itself (its rows, as
    [N, O]), which is then updated in place, but not overlap it otherwise."""
    return _C.fp8_linear(x, x_scales, weight, weight_scales, out_dtype, out, bias, activation, residual)
