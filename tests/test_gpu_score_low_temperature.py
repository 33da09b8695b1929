"""Log-probabilities of lists at the lowest temperatures that the documentation allows, masked logits and
equal largest ones among them, forward and backward, in 64 bits.

The reference takes every logit's distance to its row's maximum in 64 bits before the factor, so that a low
temperature costs it nothing.  Tolerances (e = 2^-24): forward as in test_gpu_score.  Gradient: half a
step of its type and 2e-5 of the size of its terms, as there; below |lse| = 2^31 the saved lse is two fp32
numbers and the distances are fp32, each right to 2^-24 of the first one's rounding, which is at most
2^-24 |lse|: four such errors, 2^-46 |lse|, in the exponent and in the entropy's factor.  (From 2^31 on
the values beside the maximum have probability 0 and the maximum's are equal, which is exact.)
"""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def scale_of(temperature):
    return torch.tensor(1.0 / temperature, dtype=torch.float64).float().double().item()


def reference(x, temperature):
    """(lse, entropy, log p, log p of masked logits too: by their own values) in 64 bits."""
    s, x = scale_of(temperature), x.double()
    top = x.amax(-1, keepdim=True)
    far = (x - top) * s
    d = torch.where(x <= -9.9e37, -torch.inf, far)
    log_z = d.exp().sum(-1, keepdim=True).log()
    logp = d - log_z
    p = logp.exp()
    return (top * s + log_z)[:, 0], -torch.where(p > 0, p * logp, 0.0).sum(-1), logp, far - log_z


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~((err <= tol) | (got.double() == want))
    assert not bad.any(), (what, got[bad][:4].tolist(), want[bad][:4].tolist(), int(bad.sum()))


def check(x, ids, temperature, g, g_entropy, g_lse):
    """Forward and gradient of the log-probabilities of `ids` (and of the 3 most likely tokens)."""
    leaf = x.clone().requires_grad_(True)
    lp, entropy, lse = kernel_opt.fused_token_logprobs(leaf, ids, temperature)
    lse0, h0, logp, raw = reference(x, temperature)
    want = raw.gather(1, ids)
    close(lp, want.float().double(), 1e-5 + E * want.abs().clamp(max=3e38), "logprobs")
    close(lse, lse0, 1e-5 + E * lse0.abs(), "lse")
    close(entropy, h0, 1e-5 * (1 + 3 * h0), "entropy")
    _, entropy2, lse2, top_ids, top = kernel_opt.fused_top_logprobs(x, None, 3, temperature)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :3]
    assert torch.equal(top_ids, order) and torch.equal(entropy2, entropy.detach()) and torch.equal(lse2, lse.detach())
    want = raw.gather(1, order)
    close(top, want.float().double(), 1e-5 + E * want.abs().clamp(max=3e38), "top")

    d, = torch.autograd.grad((lp, entropy, lse), leaf, (g, g_entropy, g_lse))
    p = logp.exp()
    along = torch.where(p > 0, logp, 0.0)
    gi, ge, gl = g.double(), g_entropy.double()[:, None], g_lse.double()[:, None]
    want = p * (gl - gi.sum(1, keepdim=True) - ge * (along + h0[:, None]))
    factor = gl.abs() + gi.abs().sum(1, keepdim=True) + ge.abs() * (along.abs() + h0[:, None])
    size = (p * factor).scatter_add(1, ids, gi.abs())
    want = want.scatter_add(1, ids, gi)
    s = scale_of(temperature)
    rest = 2.0 ** -46 * lse0.abs()[:, None]
    rest = torch.where(lse0.abs()[:, None] < 2.0 ** 31, rest, 0.0) * p * (factor + ge.abs())
    tol = U[x.dtype] * (s * want).abs() + s * (2e-5 * size + rest) + TINY[x.dtype] + 2.0 ** -126 * s * factor
    got = d.double()
    over = (s * want).abs() > torch.finfo(x.dtype).max  # rounds to infinity
    bad = ~(((got - s * want).abs() <= tol) | (over & (got.abs() >= torch.finfo(x.dtype).max)))
    assert not bad.any(), ("gradient", got[bad][:4].tolist(), (s * want)[bad][:4].tolist(), int(bad.sum()))


def upstream(n, k, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: size * torch.randn(s, generator=g, device="cuda")
    return r(n, k), r(n), r(n)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v", [(6, 1003), (6, 40001), (900, 5003)])
@pytest.mark.parametrize("temperature", [1e-3, 1e-6, 1e-8, 2e-9, 1e-9, 1e-12, 1e-20, 1e-30])
def test_low_temperatures(dtype, n, v, temperature):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (3 * torch.randn(n, v, generator=g, device="cuda")).to(dtype)
    x[0, 5:9] = x[0].max()                     # equal largest ones share the mass
    x[1, ::3] = -torch.inf
    x[2, v // 2:] = torch.finfo(dtype).min
    x[3] -= 20.0                               # all below 0
    x[4] = -x[4].abs()
    x[4, ::7] = 0.0                            # the largest is 0
    x[5] = -torch.inf
    x[5, v // 2] = 2.0
    ids = torch.randint(0, v, (n, 5), generator=g, device="cuda")
    ids[:, 0] = x.float().argmax(1)
    check(x, ids, temperature, *upstream(n, 5))
    check(x, ids, temperature, *upstream(n, 5, size=temperature))


@pytest.mark.parametrize("n,v", [(4, 1003), (900, 2000)])
def test_lse_beyond_fp32(n, v):
    x = 1e10 * torch.randn(n, v, device="cuda")
    x[0, 3:6] = x[0].max()
    ids = x.argmax(1)[:, None]
    leaf = x.clone().requires_grad_(True)
    lp, entropy, lse = kernel_opt.fused_token_logprobs(leaf, ids, 1e-30)
    _, h0, _, raw = reference(x, 1e-30)
    assert (lse.detach().abs() == torch.inf).all()
    close(lp, raw.gather(1, ids), 1e-5, "logprobs")
    close(entropy, h0, 1e-5 * (1 + 3 * h0), "entropy")
    d, = torch.autograd.grad(lp.sum() + entropy.sum(), leaf)
    assert d.isnan().all()
