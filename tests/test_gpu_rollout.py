"""The operators of a decoding step's tail together: RolloutHead against its parts in plain
torch, in a CUDA graph, and beside the training side that scores what it draws."""
import os
import sys

import pytest
import torch

import kernel_opt
from conftest import REPO

pytestmark = pytest.mark.gpu


def weights(v, h, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    return (1 + 0.1 * r(h)).to(dtype), (r(v, h) * 3 * h ** -0.5).to(dtype)


@pytest.mark.parametrize("n,h,v", [(1, 3584, 32000), (5, 272, 1003), (70, 1024, 4097)])
def test_step_is_its_parts(n, h, v):
    nw, w = weights(v, h)
    head = kernel_opt.RolloutHead(nw, w)
    x, r = torch.randn(2, n, h, device="cuda").bfloat16()
    u = torch.rand(n, device="cuda")
    q, s, _ = kernel_opt.fused_residual_rmsnorm_fp8(x, r, nw, 1e-6)
    z = kernel_opt.fp8_linear(q, s, head.weight, head.weight_scales)
    want = kernel_opt.sample_tokens(z, u, 0.8, 20, 0.95, 0.01)
    got = head.step(x, r, u, 0.8, 20, 0.95, 0.01)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # logits near the product of the unquantised operands: each operand errs by 2^-4 of an
    # element at most (and 2^-10 of its block's largest / 448 * 448), bf16 by 2^-8
    st = (x.float() + r.float()).bfloat16().double()
    y = st / (st.square().mean(1, keepdim=True) + 1e-6).sqrt() * nw.double()
    ref = y @ w.double().t()
    size = (y.abs() + y.abs().amax() * 2 ** -10) @ (w.double().abs() + w.double().abs().amax() * 2 ** -10).t()
    assert ((z.double() - ref).abs() <= (2 * 2 ** -4 + 2 ** -8) * size + 2 ** -8 * ref.abs()).all()


def test_captured_step():
    nw, w = weights(32000, 512)
    head = kernel_opt.RolloutHead(nw, w)
    x, r = torch.randn(2, 8, 512, device="cuda").bfloat16()
    u = torch.rand(8, device="cuda")
    head.step(x, r, u, top_p=0.9)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = head.step(x, r, u, top_p=0.9)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        u.copy_(torch.rand_like(u))
        g.replay()
        want = head.step(x, r, u, top_p=0.9)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_update_takes_new_weights():
    nw, w = weights(1000, 256)
    nw2, w2 = weights(1000, 256, seed=1)
    head = kernel_opt.RolloutHead(nw, w)
    x = torch.randn(3, 256, device="cuda").bfloat16()
    head.update(nw2, w2)
    assert torch.equal(head.logits(x), kernel_opt.RolloutHead(nw2, w2).logits(x))


def test_update_reaches_captured_steps():
    nw, w = weights(1000, 256)
    nw2, w2 = weights(1000, 256, seed=1)
    head = kernel_opt.RolloutHead(nw, w)
    x = torch.randn(3, 256, device="cuda").bfloat16()
    want = head.logits(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = head.logits(x)
    nw.copy_(nw2)  # as an optimizer writes it: the head keeps both weights until it is told
    assert torch.equal(head.logits(x), want)
    head.update(nw2, w2)
    g.replay()
    assert torch.equal(out, kernel_opt.RolloutHead(nw2, w2).logits(x))


def test_refusals():
    nw, w = weights(100, 64)
    with pytest.raises(ValueError, match="norm_weight"):
        kernel_opt.RolloutHead(nw[:32], w)
    head = kernel_opt.RolloutHead(nw, w)
    with pytest.raises(ValueError, match="one value per column"):
        head.logits(torch.zeros(2, 32, device="cuda", dtype=torch.bfloat16))


def test_example_scores_its_rollout():
    sys.path.insert(0, os.path.join(REPO, "examples"))
    from rollout_head import rollout
    out = rollout(batch=16, steps=3, hidden=512, vocab=4096)
    assert out["tokens"].shape == (3, 16) and (out["tokens"] >= 0).all()
    # the same policy but for the 8-bit operands: log-probabilities a little apart, and on
    # average hardly (the operands' rounding errors are independent of the token drawn)
    gap = out["new"] - out["old"]
    assert gap.abs().max() < 1.0 and gap.mean().abs() < 0.1
    assert all(g is not None and torch.isfinite(g).all() for g in out["grads"])
