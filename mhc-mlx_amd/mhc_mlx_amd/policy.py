"""Clipped policy loss with a KL term, from a model's logits.

For a token with logits z, action a, advantage A, and the log probabilities ``old`` (of the policy that acted) and
``ref`` (of the reference policy):

    lp = log_softmax(z)[a];  r = exp(lp - old);  q = exp(ref - lp)
    L  = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (q - 1 - log q)
    loss = sum w L / D,   D = denominator, or the sum of the weights (1 if that is 0)

Tokens of weight 0 (a prompt, padding) are left out whatever their logits, action or other inputs hold, NaN and -100
among them: they add nothing to the loss, their log probability is given as 0 and their gradient is 0.  An action
outside [0, V) of a token that counts makes the loss and that token's gradient NaN (it cannot be refused without
waiting for the GPU).

``policy_loss`` is differentiable in the logits; ``policy_loss_and_grad`` returns the gradient with the loss and reads
the logits from memory once, for a caller that continues with ``logits.backward(dlogits)``.
"""

from __future__ import annotations

import torch

from . import ops
from .profiling import timed

__all__ = ["policy_loss", "policy_loss_and_grad"]


def _check(clip_low, clip_high, denominator) -> float:
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"clip_low and clip_high must be >= 0 (got {clip_low}, {clip_high})")
    if denominator is not None and not denominator > 0:
        raise ValueError(f"denominator must be positive (got {denominator})")
    return 0.0 if denominator is None else float(denominator)


class PolicyLossFn(torch.autograd.Function):
    """policy_loss with its host steps in Python: under a kernel timer, and for torch.jit.trace, which records it."""

    @staticmethod
    def forward(ctx, logits, actions, old_logp, advantages, ref_logp, mask, *numbers):
        with timed("policy_loss_fwd"):
            loss, logp, stats = ops._binding().policy_fwd(logits, actions, old_logp, advantages, ref_logp, mask, *numbers)
        ctx.save_for_backward(logits, actions, old_logp, advantages, ref_logp, mask, stats)
        ctx.numbers = numbers
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _dlogp):
        if dloss is None:
            return (None,) * 10
        *tensors, stats = ctx.saved_tensors
        with timed("policy_loss_bwd"):
            dlogits = ops._binding().policy_bwd(*tensors, *ctx.numbers, stats, dloss)
        return (dlogits,) + (None,) * 9


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, denominator: float | None = None):
    """(loss, logp): the scalar loss, differentiable in ``logits``, and each token's log probability (no gradient).

    logits [..., V] float32, bfloat16 or float16; the others [...]: actions int64 or int32, old_logp, advantages and
    ref_logp floating, mask bool, uint8 or floating weights.  Without ref_logp, or with kl_coef 0, there is no KL term.
    """
    den = _check(clip_low, clip_high, denominator)
    numbers = float(clip_low), float(clip_high), float(kl_coef), den
    if ops._use_binding() and torch.autograd.forward_ad._current_level < 0:  # (forward mode is refused by the Function)
        return ops._binding().policy_loss(logits, actions, old_logp, advantages, ref_logp, mask, *numbers)
    return PolicyLossFn.apply(logits, actions, old_logp, advantages, ref_logp, mask, *numbers)


@torch.no_grad()
def policy_loss_and_grad(logits: torch.Tensor, actions: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                         ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                         clip_high: float = 0.2, kl_coef: float = 0.0, denominator: float | None = None,
                         grad_scale: float = 1.0):
    """(loss, logp, dlogits): policy_loss and grad_scale times its gradient, in the logits' dtype, in one call. No autograd.

    ``grad_scale`` is the loss scale of float16 training (the loss itself is not scaled).
    """
    den = _check(clip_low, clip_high, denominator)
    with timed("policy_loss_and_grad"):
        return ops._binding().policy_loss_and_grad(logits, actions, old_logp, advantages, ref_logp, mask, float(clip_low),
                                                   float(clip_high), float(kl_coef), den, float(grad_scale))
