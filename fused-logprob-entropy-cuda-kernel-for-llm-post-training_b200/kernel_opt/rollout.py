"""The tail of a decoding step in one object: final norm, 8-bit LM head, sampled token.

    stream = x + residual;  h = RMS norm(stream) in 8 bits      (kernel_opt.norm)
    logits = h W^T (+ bias), W in 8 bits with a scale per 128 x 128   (kernel_opt.fp8)
    token, log-probabilities                                    (kernel_opt.sampling)
    the most likely alternatives, where asked for               (kernel_opt.score)

With a `post_norm_weight` (models that also normalise a block's output) the stream is residual_scale *
residual + branch_scale * gate * norm(x), in the same kernel.  Three kernels a step; the logits are
written once and read once (and once more for alternatives).  The weight is quantised
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
from .norm import fused_residual_rmsnorm_fp8, fused_sandwich_rmsnorm_fp8
from .sampling import sample_tokens
from .score import fused_top_logprobs


class RolloutHead:
    """norm_weight: [H]; lm_head_weight: [V, H] bf16 / fp16 / fp32, H a multiple of 16.

    `logits_dtype`: what the product is rounded to before sampling.  bf16 (the default) is
    the rounding of the training head (`fused_linear_logprob_entropy`).

    post_norm_weight: [H] like norm_weight, for models with a norm after the last block (x is that
    block's output then, and every call needs the residual); branch_scale, residual_scale: as in
    `fused_sandwich_rmsnorm`; lm_head_bias: [V] of logits_dtype or fp32."""

    def __init__(self, norm_weight: torch.Tensor, lm_head_weight: torch.Tensor, eps: float = 1e-6,
                 logits_dtype: torch.dtype = torch.bfloat16, post_norm_weight: torch.Tensor | None = None,
                 branch_scale: float = 1.0, residual_scale: float = 1.0,
                 lm_head_bias: torch.Tensor | None = None):
        if lm_head_weight.dim() != 2 or norm_weight.shape != lm_head_weight.shape[1:]:
            raise ValueError(f"norm_weight [H] and lm_head_weight [V, H] expected, got "
                             f"{tuple(norm_weight.shape)} and {tuple(lm_head_weight.shape)}")
        if post_norm_weight is None and (branch_scale != 1.0 or residual_scale != 1.0):
            raise ValueError("branch_scale and residual_scale go with a post_norm_weight")
        self.eps = eps
        self.logits_dtype = logits_dtype
        self.branch_scale, self.residual_scale = branch_scale, residual_scale
        self.norm_weight = self.weight = self.weight_scales = self.post_norm_weight = self.bias = None
        self._has = (post_norm_weight is not None, lm_head_bias is not None)
        self.update(norm_weight, lm_head_weight, post_norm_weight, lm_head_bias)

    def update(self, norm_weight: torch.Tensor, lm_head_weight: torch.Tensor,
               post_norm_weight: torch.Tensor | None = None, lm_head_bias: torch.Tensor | None = None) -> None:
        """Take (and quantise) new weights: those that the head was built with.  All are copies: a step
        sees the weights of the last update.  They are written where the old ones of the same shape and
        type lie, so captured steps see them too."""
        if (post_norm_weight is not None, lm_head_bias is not None) != self._has:
            raise ValueError("update takes the weights that the head was built with: post_norm_weight "
                             f"{'expected' if self._has[0] else 'not expected'}, lm_head_bias "
                             f"{'expected' if self._has[1] else 'not expected'}")
        if post_norm_weight is not None and post_norm_weight.shape != norm_weight.shape:
            raise ValueError(f"post_norm_weight must be shaped like norm_weight {tuple(norm_weight.shape)}, got "
                             f"{tuple(post_norm_weight.shape)}")
        if lm_head_bias is not None and lm_head_bias.shape != lm_head_weight.shape[:1]:
            raise ValueError(f"lm_head_bias must be [V] for lm_head_weight {tuple(lm_head_weight.shape)}, got "
                             f"{tuple(lm_head_bias.shape)}")
        if lm_head_bias is not None and lm_head_bias.dtype not in (self.logits_dtype, torch.float32):
            raise ValueError(f"lm_head_bias must be {self.logits_dtype} or float32, got {lm_head_bias.dtype}")
        names = ["norm_weight", "weight", "weight_scales", "post_norm_weight", "bias"]
        new = [norm_weight.detach(), *quantize_fp8_blocks(lm_head_weight.detach()),
               *(None if t is None else t.detach() for t in (post_norm_weight, lm_head_bias))]
        old = [getattr(self, n) for n in names]
        if old[0] is not None and all((a is None) == (b is None) and (a is None or (
                a.shape == b.shape and a.dtype == b.dtype and a.device == b.device)) for a, b in zip(old, new)):
            for a, b in zip(old, new):
                if a is not None:
                    a.copy_(b)
        else:
            for i, (n, b) in enumerate(zip(names, new)):
                setattr(self, n, b if b is None or i in (1, 2) else b.clone())

    def logits(self, x: torch.Tensor, residual: torch.Tensor | None = None,
               gate: torch.Tensor | None = None) -> torch.Tensor:
        """[..., V] logits of the last layer's output x [..., H] and the residual stream (and, with a
        post_norm_weight, the block's gate: see `fused_sandwich_rmsnorm`)."""
        if self.post_norm_weight is None:
            if gate is not None:
                raise ValueError("a gate goes with a post_norm_weight")
            q, scales, _ = fused_residual_rmsnorm_fp8(x, residual, self.norm_weight, self.eps)
        else:
            if residual is None:
                raise ValueError("a head with a post_norm_weight needs the residual")
            q, scales, _ = fused_sandwich_rmsnorm_fp8(x, residual, self.post_norm_weight, self.norm_weight, gate,
                                                      self.branch_scale, self.residual_scale, self.eps)
        return fp8_linear(q, scales, self.weight, self.weight_scales, self.logits_dtype, bias=self.bias)

    def step(self, x: torch.Tensor, residual: torch.Tensor | None, u: torch.Tensor, temperature=1.0,
             top_k=0, top_p=1.0, min_p=0.0, gate: torch.Tensor | None = None):
        """(tokens, logprobs, kept_logprobs) of `sample_tokens`, each shaped like u: one token per
        row of x [..., H] from the uniform random numbers u [...]."""
        return sample_tokens(self.logits(x, residual, gate), u, temperature, top_k, top_p, min_p)

    def step_with_top(self, x: torch.Tensor, residual: torch.Tensor | None, u: torch.Tensor, k: int,
                      temperature: float = 1.0, top_k=0, top_p=1.0, min_p=0.0, gate: torch.Tensor | None = None):
        """(tokens, logprobs, kept_logprobs, entropy, top_ids, top_logprobs): `step`, with the whole
        distribution's entropy and its k most likely tokens (`fused_top_logprobs`) at the same temperature
        (at 0: at 1, as for logprobs), which is one number for all rows."""
        if isinstance(temperature, torch.Tensor):
            raise ValueError("step_with_top takes one temperature for all rows")
        logits = self.logits(x, residual, gate)
        drawn = sample_tokens(logits, u, temperature, top_k, top_p, min_p)
        _, entropy, _, ids, top = fused_top_logprobs(logits, None, k, temperature if temperature != 0 else 1.0)
        return (*drawn, entropy, ids, top)
