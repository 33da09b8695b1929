"""Sample a rollout's tokens with the 8-bit decoding head, then score them as training does.

A random head over random hidden states stands in for a model's: for every step of a rollout
the decoding head (final norm, 8-bit LM head, sampling) draws one token per sequence; the
same hidden states then go through the training side (norm in bf16, LM head fused with K1),
with gradients.  Prints how far the two log-probabilities of the drawn tokens are apart (the
log of GRPO's ratio before any update) and the step's time.

    python examples/rollout_head.py [--batch 64 --steps 16 --hidden 3584 --vocab 151936]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "fused-logprob-entropy-cuda-kernel-for-llm-post-training_b200"))
import kernel_opt  # noqa: E402


def rollout(batch, steps, hidden, vocab, temperature=1.0, top_p=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    norm_weight = (1 + 0.1 * normal(hidden)).requires_grad_(True)
    head_weight = (normal(vocab, hidden) * 3.0 * hidden ** -0.5).requires_grad_(True)
    head = kernel_opt.RolloutHead(norm_weight, head_weight)

    xs, residuals, tokens, logprobs = [], [], [], []
    for _ in range(steps):
        x, residual = normal(batch, hidden), normal(batch, hidden)
        u = torch.rand(batch, generator=g, device="cuda")
        token, logprob, _ = head.step(x, residual, u, temperature=temperature, top_p=top_p)
        for keep, value in zip((xs, residuals, tokens, logprobs), (x, residual, token, logprob)):
            keep.append(value)
    x, residual, token, old = (torch.stack(v) for v in (xs, residuals, tokens, logprobs))

    # the training side, on the same states
    h, _ = kernel_opt.fused_residual_rmsnorm(x, residual, norm_weight)
    new, _, _ = kernel_opt.fused_linear_logprob_entropy(h, head_weight, token, temperature)
    ratio = (new - old).exp()
    (-ratio.mean()).backward()
    return {"tokens": token, "old": old, "new": new.detach(), "head": head,
            "grads": (norm_weight.grad, head_weight.grad)}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--hidden", type=int, default=3584)
    ap.add_argument("--vocab", type=int, default=151936)
    a = ap.parse_args()
    out = rollout(a.batch, a.steps, a.hidden, a.vocab)
    gap = (out["new"] - out["old"]).abs()
    print(f"{a.steps} steps of {a.batch} sequences: |log ratio| mean {gap.mean():.4f}, max {gap.max():.4f}")

    x = torch.randn(a.batch, a.hidden, device="cuda").bfloat16()
    u = torch.rand(a.batch, device="cuda")
    for _ in range(3):
        out["head"].step(x, x, u)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(20):
        out["head"].step(x, x, u)
    end.record()
    end.synchronize()
    print(f"one decoding step's tail: {start.elapsed_time(end) / 20 * 1e3:.1f} us")


if __name__ == "__main__":
    main()
