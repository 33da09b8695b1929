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

from .norm import _rows

OUT_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def quantize_fp8_rows(x: torch.Tensor):
    """(q, scales) of x [..., H] (bf16 / fp16 / fp32, H at most 16384): q float8_e4m3fn like x,
    scales fp32 [..., ceil(H / 128)]; x is about q * scale."""
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    q, scales = _C.quantize_fp8_rows(_rows(x))
    return q.view(x.shape), scales.view(*x.shape[:-1], scales.shape[-1])


def quantize_fp8_blocks(weight: torch.Tensor):
    """(q, scales) of a weight [O, H]: q float8_e4m3fn [O, H], scales fp32
    [ceil(O / 128), ceil(H / 128)]."""
    if not weight.is_cuda or weight.dim() != 2:
        raise ValueError("weight must be a CUDA tensor [O, H]")
    return tuple(_C.quantize_fp8_blocks(weight if weight.stride(1) == 1 else weight.contiguous()))


def fp8_linear(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor,
               weight_scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """(x * x_scales) @ (weight * weight_scales).T: [..., O] in `out_dtype` (bf16 / fp16 / fp32).

    x: float8_e4m3fn [..., H]; x_scales: fp32 [..., ceil(H / 128)]; weight: float8_e4m3fn
    [O, H]; weight_scales: fp32 [ceil(O / 128), ceil(H / 128)].  H must be a multiple of 16, at
    most 32768.  `out`: a tensor to write ([N, O], unit stride along O) instead of a new one."""
    if out_dtype not in OUT_DTYPES and out is None:
        raise ValueError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
    lead = x.shape[:-1]
    x2 = _rows(x)
    if x_scales.shape[:-1] != lead:
        raise ValueError(f"x_scales must have x's leading dimensions {tuple(lead)}, got "
                         f"{tuple(x_scales.shape)}")
    y = out if out is not None else torch.empty((x2.shape[0], weight.shape[0]), dtype=out_dtype,
                                                device=x.device)
    _C.fp8_linear(x2, x_scales.reshape(-1, x_scales.shape[-1]).contiguous(), weight,
                  weight_scales.contiguous(), y)
    return y if out is not None else y.view(*lead, weight.shape[0])
