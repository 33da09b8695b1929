"""Tokens from logits, with temperature, top-k, top-p and min-p and given random numbers.

One kernel over the rows of [..., V] logits (csrc/k1_sample.cuh), which reads them once.  The
random numbers are inputs, and the sums that decide a token are right to about 1e-12 of the mass,
so the same logits and numbers give the same token whatever batch the row is in, unless a number
lies that close to the boundary between two tokens.  The returned `logprob` is K1's log-probability
of the drawn token under the logits given (at the sampling temperature, over the whole vocabulary).
It is the old-policy value of GRPO's ratio where those are the training head's logits; an 8-bit
head's are another policy's (see `kernel_opt.rollout`).  No counterpart in the reference, whose
generation runs in another library.
"""
from __future__ import annotations

import torch

from kernel_opt import _C


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0):
    """(tokens, logprobs, kept_logprobs), each shaped like `u`.

    logits: [..., V] bf16 / fp16 / fp32; u: [...] fp32 in [0, 1).  temperature, top_k, top_p,
    min_p: numbers, or tensors shaped like u (one setting per row).

    Logits are divided by the temperature (multiplied by fp32(1/T)); top-k keeps the k most
    likely tokens (the lower id among equals), top-p the shortest prefix of those with at
    least that share of their probability, min-p those at least min_p times as likely as the
    first; the first always stays.  The token is the first kept id at which the kept
    probability up to it, in the order of ids, exceeds u.  top_k <= 0, top_p >= 1 and min_p = 0
    are off; temperature 0 takes the first largest logit.

    logprobs: of the token in the whole distribution at this temperature (at 0: at 1);
    kept_logprobs: in the filtered, renormalised one.  No gradient flows.  A row with a NaN or
    +inf (after the division too), or nothing above -inf, gives token -1 and NaN; so does one whose
    own setting means nothing (a temperature that is negative or not finite, a negative top_p, a
    min_p outside [0, 1], a NaN), which as a number for all rows is refused."""
    return _C.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
