"""Residual addition + root-mean-square norm, for training and with an output in 8 bits.

    stream = x + residual            rounded to the tensors' dtype and stored
    y      = stream * rstd * weight  rstd = 1 / sqrt(mean(stream^2) + eps), fp32 per row

The norm reads the stream as it is stored, so it equals an addition followed by a norm, and
the backward (which keeps the stream and rstd) and the next layer see the same numbers.  One
kernel each way over rows of bf16 / fp16 / fp32; sums and the weight's gradient are fp32, the
latter added in a fixed order.  No counterpart in the reference.
"""
from __future__ import annotations

import torch

from kernel_opt import _C


def fused_residual_rmsnorm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                           eps: float = 1e-6):
    """(y, stream): stream = x + residual, y = RMS norm of the stream times `weight`.

    x, residual: [..., H] bf16 / fp16 / fp32 of one shape and dtype (H at most 16384; rows may
    be strided); weight: [H] of the same dtype or fp32.  `residual=None`: stream is x itself.
    Differentiable (once, backwards) in x, residual and weight, through y and through the stream."""
    return _C.residual_rmsnorm(x, residual, weight, eps)


def fused_residual_rmsnorm_fp8(x: torch.Tensor, residual: torch.Tensor | None,
                               weight: torch.Tensor, eps: float = 1e-6):
    """(q, scales, stream): `fused_residual_rmsnorm` with y in 8 bits, for `fp8_linear`.

    q: float8_e4m3fn like x; scales: fp32 [..., ceil(H / 128)], one per row and 128 columns
    (largest magnitude / 448), y = q * scale.  y is rounded once, from fp32.  Inference only:
    no gradient flows."""
    return _C.residual_rmsnorm_fp8(x, residual, weight, eps)
