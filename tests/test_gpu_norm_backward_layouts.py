"""Gradients of the residual RMS norm that arrive in rows of any pitch and start: the backward's
vector, pair and single-element paths, chosen by address and pitch instead of by width."""
import pytest
import torch

import kernel_opt
from test_gpu_norm import DTYPES, EPS, check_grads, inputs

pytestmark = pytest.mark.gpu


def laid_out(t, off, pitch):
    """t's values in rows `pitch` elements apart that start `off` elements after a vector boundary."""
    n, h = t.shape
    wide = torch.full((n, pitch), float("nan"), dtype=t.dtype, device="cuda")
    view = wide[:, off:off + h]
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["gy", "gs", "both", "stream"])
@pytest.mark.parametrize("n,h", [(37, 384), (300, 1026), (5, 513), (2, 8192)])
def test_strided_gradients(n, h, which, dtype):
    x, r, w, gy, gs = inputs(n, h, dtype)
    for off, pad in ((0, 8), (8, 16), (2, 6), (1, 3), (1, 8), (0, 1)):
        lay = lambda t, on: laid_out(t, off, h + off + pad) if on else t
        if which == "stream":   # without a residual the stream is x itself, in its own layout
            a = lay(x, True).requires_grad_(True)
            b = w.clone().requires_grad_(True)
            y, s = kernel_opt.fused_residual_rmsnorm(a, None, b, EPS)
            dx, dw = torch.autograd.grad(y, (a, b), gy)
            check_grads(gy, None, x, w, dx, dw)
            continue
        a, c, b = (t.clone().requires_grad_(True) for t in (x, r, w))
        y, s = kernel_opt.fused_residual_rmsnorm(a, c, b, EPS)
        dx, dr, dw = torch.autograd.grad((y, s), (a, c, b), (lay(gy, which != "gs"), lay(gs, which != "gy")))
        assert torch.equal(dx, dr)
        check_grads(gy, gs, s.detach(), w, dx, dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_gradient_that_every_row_shares(dtype):
    """Broadcast over the rows (a pitch of 0), and transposed (no unit stride)."""
    n, h = 40, 256
    x, r, w, gy, gs = inputs(n, h, dtype)
    a, c, b = (t.clone().requires_grad_(True) for t in (x, r, w))
    y, s = kernel_opt.fused_residual_rmsnorm(a, c, b, EPS)
    one = gy[:1].expand(n, h)
    turned = gs.t().contiguous().t()
    dx, _, dw = torch.autograd.grad((y, s), (a, c, b), (one, turned))
    check_grads(one, gs, s.detach(), w, dx, dw)


def test_a_weight_off_a_vector_boundary():
    for dtype, wdtype in ((torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)):
        x, r, w, gy, gs = inputs(33, 520, dtype, wdtype)
        for off in (1, 2, 4):
            buf = torch.zeros(520 + off, dtype=wdtype, device="cuda")
            view = buf[off:]
            view.copy_(w)
            a, c = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
            b = view.requires_grad_(True)
            y, s = kernel_opt.fused_residual_rmsnorm(a, c, b, EPS)
            dx, _, dw = torch.autograd.grad((y, s), (a, c, b), (gy, gs))
            check_grads(gy, gs, s.detach(), w, dx, dw)
