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


def fused_sandwich_rmsnorm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                           weight: torch.Tensor, gate: torch.Tensor | None = None,
                           branch_scale: float = 1.0, residual_scale: float = 1.0, eps: float = 1e-6):
    """(y, stream): the norm after a block and the one before the next.

        stream = residual_scale * residual + branch_scale * gate * (RMS norm of x times post_weight)
        y      = RMS norm of the stream (as stored) times weight

    x, residual: [..., H] as in `fused_residual_rmsnorm`; post_weight, weight: [H] of x's dtype or
    both fp32.  gate: None, [H] of the weights' dtype, or x's leading dimensions with H or 1 columns in
    x's dtype (other shapes: expand them; beside a single row [H] its dtype says which it is).  branch_scale, residual_scale: finite numbers.
    Differentiable (once, backwards) in x, residual, both weights and the gate, through y and the
    stream.  Rows of few and of many (more than the device has SMs) are summed in different orders,
    so a row's last bits may depend on which of the two it is in; within either they do not depend
    on the other rows, and the same call gives the same bits."""
    return _C.sandwich_rmsnorm(x, residual, post_weight, weight, gate, branch_scale, residual_scale, eps)


def fused_sandwich_rmsnorm_fp8(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                               weight: torch.Tensor, gate: torch.Tensor | None = None,
                               branch_scale: float = 1.0, residual_scale: float = 1.0, eps: float = 1e-6):
    """(q, scales, stream): `fused_sandwich_rmsnorm` with y in 8 bits, for `fp8_linear` (q and
    scales as in `fused_residual_rmsnorm_fp8`).  Inference only: no gradient flows."""
    return _C.sandwich_rmsnorm_fp8(x, residual, post_weight, weight, gate, branch_scale, residual_scale, eps)
