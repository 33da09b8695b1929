"""Forward-mode differentiation of the residual RMS norm is refused, as K1's functions refuse it: a
tangent is not dropped without a word, whether the inputs also require a gradient or not."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import kernel_opt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dual", ["x", "residual", "weight"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(dual, requires_grad):
    ins = {"x": torch.randn(3, 64, device="cuda"), "residual": torch.randn(3, 64, device="cuda"),
           "weight": torch.ones(64, device="cuda")}
    ins = {k: v.requires_grad_(requires_grad) for k, v in ins.items()}
    with fwd.dual_level():
        with_tangent = dict(ins)
        with_tangent[dual] = fwd.make_dual(ins[dual], torch.ones_like(ins[dual]))
        with pytest.raises(RuntimeError, match="forward AD"):
            kernel_opt.fused_residual_rmsnorm(**with_tangent)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward AD"):
            kernel_opt.fused_residual_rmsnorm(**with_tangent)
        kernel_opt.fused_residual_rmsnorm(**ins)   # no tangent
        if dual != "residual":
            with pytest.raises(RuntimeError, match="forward AD"):
                kernel_opt.fused_residual_rmsnorm(with_tangent["x"], None, with_tangent["weight"])
