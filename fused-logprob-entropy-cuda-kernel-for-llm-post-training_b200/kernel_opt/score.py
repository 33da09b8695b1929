"""Log-probabilities with alternatives: of K given tokens, and of the k most likely ones.

K1 scores one target per position.  Rollouts, evaluation and distillation also ask for the most
likely tokens of a position (a teacher's list, a client's alternatives) and for the
log-probabilities of a given list (a student on that list).  One kernel reads the logits once and
returns them with entropy and log-sum-exp; one reads them once more and writes their gradient
(csrc/k1_score.cuh).

A temperature T means y = x * fp32(1 / T), not rounded to the logits' type, as in
`kernel_opt.sampling` (`fused_logprob_entropy_scaled` rounds it as an in-place division would).
No counterpart in the reference.
"""
from __future__ import annotations

import torch

from kernel_opt import _C


def fused_top_logprobs(logits: torch.Tensor, targets: torch.Tensor | None, k: int, temperature: float = 1.0):
    """(logprob, entropy, lse, top_ids, top_logprobs) of logits / temperature.

    logits: [..., V] bf16 / fp16 / fp32 (rows may be strided as in `fused_logprob_entropy`);
    targets: [...] int64 or None (logprob is None then); k: 1 to min(128, V); temperature: 1e-30 to
    1e30.  logprob, entropy, lse: [...] fp32, as `fused_logprob_entropy` returns them; top_ids:
    [..., k] int64, the largest logits first and the lowest id first among equals; top_logprobs:
    [..., k] fp32.

    Differentiable (once, backwards) in logits through all but top_ids.  Logits at or below about
    -1e38 are masked: probability 0, after all others.  A row with a NaN or +inf, or with every logit
    masked, gives ids -1 and NaN (lse -inf where all are masked).  Where a low temperature puts lse
    beyond fp32's range it is infinite and the gradient NaN.  A row whose upstream gradients are all
    zero gets a zero gradient whatever it holds."""
    return _C.top_logprobs(logits, targets, k, temperature)


def fused_token_logprobs(logits: torch.Tensor, token_ids: torch.Tensor, temperature: float = 1.0):
    """(logprobs, entropy, lse): log-probabilities of K given tokens per row of logits / temperature.

    token_ids: [..., K] int64, K at most 1024; logprobs: [..., K] fp32; entropy, lse: [...] fp32.
    An id outside [0, V) (a list's padding, say -100) reads a logit of 0, as K1's targets do: its
    log-probability is -lse and it has no gradient of its own.  A token may be named twice: it gets
    both gradients.  Otherwise as `fused_top_logprobs`."""
    return _C.token_logprobs(logits, token_ids, temperature)
