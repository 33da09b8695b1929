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


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., H] as [N, H] with unit stride inside a row; a view where the layout allows it."""
    if t.dim() == 0:
        raise ValueError("a tensor with a hidden dimension is expected")
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check(x, residual, weight, eps):
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError(f"residual must match x in shape, dtype and device, got "
                         f"{tuple(residual.shape)} {residual.dtype} for {tuple(x.shape)} {x.dtype}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must have one value per column ({x.shape[-1]}), got "
                         f"{tuple(weight.shape)}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps!r}")


class _ResidualRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        x2 = _rows(x)
        w = weight.contiguous()
        y, stream, rstd = _C.residual_rmsnorm(
            x2, None if residual is None else _rows(residual), w, eps)
        ctx.save_for_backward(stream, rstd, w)
        ctx.set_materialize_grads(False)
        y = y.view(x.shape)
        return y if residual is None else (y, stream.view(x.shape))

    @staticmethod
    def backward(ctx, g_y, g_stream=None):
        stream, rstd, weight = ctx.saved_tensors
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        if g_y is None:  # only the stream was used: the addition's own gradient
            return (g_stream if need_x else None, g_stream if need_r else None, None, None)
        d, dw = _C.residual_rmsnorm_backward(
            _rows(g_y), None if g_stream is None else _rows(g_stream), stream, rstd, weight,
            need_x or need_r, need_w)
        if d is not None:
            d = d.view(g_y.shape)
        return (d if need_x else None, d if need_r else None, dw, None)


def fused_residual_rmsnorm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                           eps: float = 1e-6):
    """(y, stream): stream = x + residual, y = RMS norm of the stream times `weight`.

    x, residual: [..., H] bf16 / fp16 / fp32 of one shape and dtype (H at most 16384; rows may
    be strided); weight: [H] of the same dtype or fp32.  `residual=None`: stream is x itself.
    Differentiable in x, residual and weight, through y and through the stream."""
    _check(x, residual, weight, eps)
    if residual is None:
        return _ResidualRMSNorm.apply(x, None, weight, float(eps)), x
    return _ResidualRMSNorm.apply(x, residual, weight, float(eps))


def fused_residual_rmsnorm_fp8(x: torch.Tensor, residual: torch.Tensor | None,
                               weight: torch.Tensor, eps: float = 1e-6):
    """(q, scales, stream): `fused_residual_rmsnorm` with y in 8 bits, for `fp8_linear`.

    q: float8_e4m3fn like x; scales: fp32 [..., ceil(H / 128)], one per row and 128 columns
    (largest magnitude / 448), y = q * scale.  y is rounded once, from fp32.  Inference only:
    no gradient flows."""
    _check(x, residual, weight, eps)
    q, scales, stream = _C.residual_rmsnorm_fp8(
        _rows(x), None if residual is None else _rows(residual), weight.contiguous(), float(eps))
    return (q.view(x.shape), scales.view(*x.shape[:-1], scales.shape[-1]),
            x if residual is None else stream.view(x.shape))
