"""The gradient of masked logits is 0 (and that of the others right) where the factor of the entropy's gradient,
s g_H, is large: low temperatures that the documentation allows, large upstream gradients."""
import pytest
import torch

import kernel_opt
from test_gpu_score import DTYPES, check_gradient, logits_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v", [(4, 1003), (3, 40000)])
@pytest.mark.parametrize("temperature,size", [(1.0, 1e12), (1e-4, 1e6), (1e-6, 1e3)])
def test_masked(dtype, n, v, temperature, size):
    x = logits_of(n, v, dtype)
    x[0, ::3] = -torch.inf
    x[1, 5:] = torch.finfo(dtype).min
    x[2, :-2] = -torch.inf
    # every row has one token with all the mass, so nothing but zeros is expected, in any type
    for r, at in enumerate((1, 2, v - 1)):
        x[r, at] = 60.0
    leaf = x.clone().requires_grad_(True)
    _, entropy, _ = kernel_opt.fused_token_logprobs(leaf, torch.zeros(n, 1, dtype=torch.int64, device="cuda"), temperature)
    d, = torch.autograd.grad(entropy[:3].sum() * size, leaf, retain_graph=True)
    masked = (x == -torch.inf) | (x == torch.finfo(dtype).min)
    assert not d.isnan().any() and (d[masked] == 0).all() and (d[3:] == 0).all()
    if temperature == 1.0:
        d, = torch.autograd.grad(entropy.sum(), leaf)
        one = torch.ones(n, device="cuda")
        check_gradient(x, d, torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.zeros(n, 1, device="cuda"), one,
                       None, 1.0)
