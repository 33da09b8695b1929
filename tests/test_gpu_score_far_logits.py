"""Log-probabilities of lists over finite logits up to the types' largest, masked ones beside them, forward
and backward, in 64 bits (checks and tolerances: test_gpu_score_low_temperature)."""
import pytest
import torch

from test_gpu_score_low_temperature import check, upstream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("n,v", [(6, 1003), (6, 40001), (900, 5003)])
@pytest.mark.parametrize("size,temperature", [(5e30, 1.0), (2e31, 1.0), (3e36, 1.0), (1e31, 1e30), (3e38, 1.0), (3e38, 1e30)])
def test_far_logits(dtype, n, v, size, temperature):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (torch.rand(n, v, generator=g, device="cuda") * 2 - 1).mul_(size).to(dtype)
    x[0, ::2] = x[0].max()                     # many equal ones
    x[1, ::3] = -torch.inf
    x[2, v // 2:] = torch.finfo(dtype).min
    x[3] = -x[3].abs()
    x[4, 1:] = -1.0
    x[4, 0] = size
    ids = torch.randint(0, v, (n, 5), generator=g, device="cuda")
    ids[:, 0] = x.float().argmax(1)
    check(x, ids, temperature, *upstream(n, 5))
