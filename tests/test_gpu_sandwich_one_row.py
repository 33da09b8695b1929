"""A single row [H] with weights in fp32 and a gate [H]: of the weights' type it is a gate per column, of the
row's type one per element, as for rows in more dimensions."""
import pytest
import torch

import kernel_opt
from test_gpu_sandwich_norm import EPS, check_forward, check_grads, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("h", [1, 7, 256, 1000])
def test_gate_of_either_type(dtype, h):
    for kind in ("column", "full"):
        t, gy, gs = inputs(1, h, dtype, kind, torch.float32)
        one = {k: v.reshape(h).requires_grad_(True) for k, v in t.items()}
        y, stream = kernel_opt.fused_sandwich_rmsnorm(**one, eps=EPS)
        got = dict(zip(one, torch.autograd.grad((y, stream), list(one.values()), (gy[0], gs[0]))))
        assert all(got[k].shape == (h,) and got[k].dtype == one[k].dtype for k in one)
        rows = {k: v.detach() for k, v in t.items()}
        check_forward(rows, y.detach()[None], stream.detach()[None], 1.0, 1.0)
        check_grads(rows, stream.detach()[None], gy, gs, {k: v.reshape(t[k].shape) for k, v in got.items()}, 1.0, 1.0)
        q, scales, s8 = kernel_opt.fused_sandwich_rmsnorm_fp8(**{k: v.detach() for k, v in one.items()}, eps=EPS)
        assert torch.equal(s8, stream.detach()) and q.shape == (h,)
