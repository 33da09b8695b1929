"""The operators around a block's end together, as they are used: a decoding step with a norm after the
block, a bias and alternatives (RolloutHead), and a distillation step on a teacher's lists."""
import os
import sys

import pytest
import torch

import kernel_opt
from conftest import REPO

sys.path.insert(0, os.path.join(REPO, "examples"))

pytestmark = pytest.mark.gpu


def weights(v, h, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    return {"norm_weight": (1 + 0.1 * r(h)).bfloat16(), "lm_head_weight": (r(v, h) * 3 * h ** -0.5).bfloat16(),
            "post_norm_weight": (1 + 0.1 * r(h)).bfloat16(), "lm_head_bias": r(v).bfloat16()}


def states(n, h, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (*torch.randn(2, n, h, generator=g, device="cuda").bfloat16(), torch.rand(n, generator=g, device="cuda"))


@pytest.mark.parametrize("n,h,v", [(1, 3584, 32000), (5, 272, 1003), (200, 1024, 4097)])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_step_with_top_is_its_parts(n, h, v, temperature):
    w = weights(v, h)
    head = kernel_opt.RolloutHead(**w, branch_scale=0.5)
    x, r, u = states(n, h)
    gate = torch.rand(n, 1, device="cuda").bfloat16()
    token, logprob, kept, entropy, ids, top = head.step_with_top(x, r, u, 7, temperature, top_p=0.9, gate=gate)
    assert all(torch.equal(a, b) for a, b in zip(head.step(x, r, u, temperature, top_p=0.9, gate=gate), (token, logprob, kept)))
    q, s, _ = kernel_opt.fused_sandwich_rmsnorm_fp8(x, r, w["post_norm_weight"], w["norm_weight"], gate, 0.5)
    z = kernel_opt.fp8_linear(q, s, head.weight, head.weight_scales, bias=w["lm_head_bias"])
    assert torch.equal(z, head.logits(x, r, gate))
    # the drawn token's log-probability is the list's where the list has it: both are right to 1e-5 and
    # their own rounding (the temperature's product, where there is one, rounds in the sampler: 2^-24 |y|)
    t = temperature or 1.0
    y = z.double() / t
    lse = torch.logsumexp(y, 1)
    assert (entropy.double() - (lse - (torch.softmax(y, 1) * y).sum(1))).abs().max() < 1e-4
    order = torch.sort(z.float(), dim=1, descending=True, stable=True).indices[:, :7]
    assert torch.equal(ids, order)
    got = torch.where(ids == token[:, None], top, 0.0).sum(1)
    there = (ids == token[:, None]).any(1)
    size = y.abs().amax(1) + lse.abs()
    assert ((got - logprob).double().abs() <= 2e-5 + 2.0 ** -22 * size)[there].all()
    if temperature == 0:
        assert torch.equal(ids[:, 0], token)


def test_captured_and_updated():
    w = weights(8000, 512)
    head = kernel_opt.RolloutHead(**w)
    x, r, u = states(8, 512)
    head.step_with_top(x, r, u, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = head.step_with_top(x, r, u, 5)
    w = weights(8000, 512, seed=7)
    head.update(**w)
    graph.replay()
    want = kernel_opt.RolloutHead(**w).step_with_top(x, r, u, 5)
    assert all(torch.equal(a, b) for a, b in zip(held, want))


def test_head_refuses():
    w = weights(64, 32)
    plain = {k: w[k] for k in ("norm_weight", "lm_head_weight")}
    x, r, u = states(2, 32)
    with pytest.raises(ValueError, match="post_norm_weight"):
        kernel_opt.RolloutHead(**plain, branch_scale=0.5)
    with pytest.raises(ValueError, match="shaped like norm_weight"):
        kernel_opt.RolloutHead(**plain, post_norm_weight=w["post_norm_weight"][:16])
    with pytest.raises(ValueError, match="lm_head_bias"):
        kernel_opt.RolloutHead(**plain, lm_head_bias=w["lm_head_bias"][:16])
    head = kernel_opt.RolloutHead(**w)
    with pytest.raises(ValueError, match="built with"):
        head.update(**plain)
    with pytest.raises(ValueError, match="residual"):
        head.step(x, None, u)
    with pytest.raises(ValueError, match="one temperature"):
        head.step_with_top(x, r, u, 3, torch.ones(2, device="cuda"))
    head = kernel_opt.RolloutHead(**plain)
    with pytest.raises(ValueError, match="gate"):
        head.logits(x, r, torch.ones(2, 1, device="cuda").bfloat16())
    with pytest.raises(ValueError, match="built with"):
        head.update(**w)


def test_distillation_example():
    """The example's gradients against the same step in 64 bits from the same weights.  The norms' output
    and the logits are bf16 tensors between the operators (2^-8 of an element each), and so are the
    gradients that go back through them; a sum over 48 tokens or 128 columns of such terms is held to
    2^-5 of its 2-norm."""
    import distill_lists as example
    tokens, hidden, vocab, k, temperature = 48, 128, 1000, 9, 2.0
    out = example.distill(tokens, hidden, vocab, k, temperature)
    p = {n: v.detach().double().requires_grad_(True) for n, v in out["params"].items()}
    x, residual = out["x"].double(), out["residual"].double()
    norm = lambda a, w: a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
    stream = residual + p["gate"] * norm(x, p["post_norm"])
    logits = norm(stream, p["norm"]) @ p["head"].t() / temperature
    logp = torch.log_softmax(logits, -1)
    entropy = -(logp.exp() * logp).sum(-1)
    loss = -(out["shares"].double() * logp.gather(-1, out["ids"])).sum(-1).mean() - 0.01 * entropy.mean()
    loss.backward()
    assert abs(float(loss) - float(out["loss"])) < 2.0 ** -6 * float(logits.abs().max())
    for n, v in p.items():
        got = out["params"][n].grad.double()
        assert (got - v.grad).norm() <= 2.0 ** -5 * v.grad.norm(), n
