"""A student learns a teacher's lists: the k most likely tokens of every position and their shares.

The teacher's logits give lists (ids and log-probabilities); a cross entropy on the renormalised
lists then takes the student's log-probabilities of the same tokens, with gradients through the norms at
the end of its last block, its head's weight and the block's gate.  Random states and weights stand in
for both models'.

    python examples/distill_lists.py [--tokens 512 --hidden 3584 --vocab 151936 --k 32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "fused-logprob-entropy-cuda-kernel-for-llm-post-training_b200"))
import kernel_opt  # noqa: E402


def teacher_lists(logits, k, temperature):
    """(ids, shares): the k most likely tokens of every row and their renormalised probabilities."""
    _, _, _, ids, top = kernel_opt.fused_top_logprobs(logits, None, k, temperature)
    return ids, torch.softmax(top, -1)


def student_loss(x, residual, params, ids, shares, temperature, entropy_weight=0.0):
    h, _ = kernel_opt.fused_sandwich_rmsnorm(x, residual, params["post_norm"], params["norm"], params["gate"])
    logits = h @ params["head"].t()
    logprobs, entropy, _ = kernel_opt.fused_token_logprobs(logits, ids, temperature)
    return -(shares * logprobs).sum(-1).mean() - entropy_weight * entropy.mean()


def distill(tokens, hidden, vocab, k, temperature=2.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    x, residual = normal(tokens, hidden), normal(tokens, hidden)
    ids, shares = teacher_lists(3 * normal(tokens, vocab), k, temperature)
    params = {"post_norm": 1 + 0.1 * normal(hidden), "norm": 1 + 0.1 * normal(hidden),
              "gate": 0.5 + 0.1 * normal(hidden), "head": normal(vocab, hidden) * hidden ** -0.5}
    params = {n: p.requires_grad_(True) for n, p in params.items()}
    loss = student_loss(x, residual, params, ids, shares, temperature, 0.01)
    loss.backward()
    return {"loss": loss.detach(), "ids": ids, "shares": shares, "x": x, "residual": residual, "params": params}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=3584)
    ap.add_argument("--vocab", type=int, default=151936)
    ap.add_argument("--k", type=int, default=32)
    a = ap.parse_args()
    out = distill(a.tokens, a.hidden, a.vocab, a.k)
    norms = {n: round(float(p.grad.float().norm()), 4) for n, p in out["params"].items()}
    print(f"cross entropy on {a.k} tokens: {float(out['loss']):.4f}; gradient norms {norms}")


if __name__ == "__main__":
    main()
