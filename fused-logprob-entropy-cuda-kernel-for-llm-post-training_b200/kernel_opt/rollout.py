"""The tail of a decoding step in one object: final norm, 8-bit LM head, sampled token.

    stream = x + residual;  h = RMS norm(stream) in 8 bits      (kernel_opt.norm)
    logits = h W^T, W in 8 bits with a scale per 128 x 128      (kernel_opt.fp8)
    token, log-probabilities                                    (kernel_opt.sampling)

Three kernels a step; the logits are written once and read once.  The weight is quantised
when the head is built (and by `update` after an optimizer step), not in a step.  A step
allocates only its outputs and is safe to capture in a CUDA graph.

The log-probabilities are the 8-bit head's, which drew the token.  The bf16 training head gives the
same token another value: for a random head (H = 3584, V = 151936) the two are 0.09 apart on average
and 0.4 at most over 1024 tokens.  A ratio whose old policy should be the training head's takes the old
values from `fused_linear_logprob_entropy` on the rollout's states, or corrects for the difference.
No counterpart in the reference, which scores tokens that another library generated.
"""
from __future__ import annotations

import torch

from .fp8 import fp8_linear, quantize_fp8_blocks
from .norm import fused_residual_rmsnorm_fp8
from .sampling import sample_tokens


class RolloutHead:
    """norm_weight: [H]; lm_head_weight: [V, H] bf16 / fp16 / fp32, H a multiple of 16.

    `logits_dtype`: what the product is rounded to before sampling.  bf16 (the default) is
    the rounding of the training head (`fused_linear_logprob_entropy`)."""

    def __init__(self, norm_weight: torch.Tensor, lm_head_weight: torch.Tensor, eps: float = 1e-6,
                 logits_dtype: torch.dtype = torch.bfloat16):
        if lm_head_weight.dim() != 2 or norm_weight.shape != lm_head_weight.shape[1:]:
            raise ValueError(f"norm_weight [H] and lm_head_weight [V, H] expected, got "
                             f"{tuple(norm_weight.shape)} and {tuple(lm_head_weight.shape)}")
        self.eps = eps
        self.logits_dtype = logits_dtype
        self.norm_weight = self.weight = self.weight_scales = None
        self.update(norm_weight, lm_head_weight)

    def update(self, norm_weight: torch.Tensor, lm_head_weight: torch.Tensor) -> None:
        """Take (and quantise) new weights.  Both are copies: a step sees the weights of the last
        update.  They are written where the old ones of the same shape and type lie, so captured
        steps see them too."""
        new = (norm_weight.detach(), *quantize_fp8_blocks(lm_head_weight.detach()))
        old = (self.norm_weight, self.weight, self.weight_scales)
        if old[0] is not None and all(a.shape == b.shape and a.dtype == b.dtype and a.device == b.device
                                      for a, b in zip(old, new)):
            for a, b in zip(old, new):
                a.copy_(b)
        else:
            self.norm_weight, self.weight, self.weight_scales = new[0].clone(), new[1], new[2]

    def logits(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        """[..., V] logits of the last layer's output x [..., H] and the residual stream."""
        q, scales, _ = fused_residual_rmsnorm_fp8(x, residual, self.norm_weight, self.eps)
        return fp8_linear(q, scales, self.weight, self.weight_scales, self.logits_dtype)

    def step(self, x: torch.Tensor, residual: torch.Tensor | None, u: torch.Tensor, temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0):
        """(tokens, logprobs, kept_logprobs) of `sample_tokens`, each shaped like u: one token per
        row of x [..., H] from the uniform random numbers u [...]."""
        return sample_tokens(self.logits(x, residual), u, temperature, top_k, top_p, min_p)
