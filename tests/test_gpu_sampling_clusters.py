"""Rows that several blocks share, in every number of blocks and with more rows than the device
holds at a time: each launch gives what the first gave, bit for bit."""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20, top_p=0.9)], ids=str)
@pytest.mark.parametrize("n,v,dtype", [(1, 152064, torch.bfloat16), (40, 60000, torch.float32), (400, 152064, torch.bfloat16),
                                       (320, 100001, torch.float32), (320, 152063, torch.float32)])
def test_launches_repeat(n, v, dtype, kw):
    g = torch.Generator(device="cuda").manual_seed(n + v)
    x = torch.randn(n, v, generator=g, device="cuda").mul_(3).to(dtype)
    u = torch.rand(n, generator=g, device="cuda")
    want = kernel_opt.sample_tokens(x, u, **kw)
    got = [kernel_opt.sample_tokens(x, u, **kw) for _ in range(20)]
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
