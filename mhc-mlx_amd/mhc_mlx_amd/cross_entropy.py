"""Softmax cross entropy over a vocabulary, from the last hidden states and the head's weight.

For a token with hidden state x and target y, and the logits z = weight x:

    logp = log_softmax(z)[y];  loss = -sum w logp / D,   D = denominator, or the sum of the weights (1 if that is 0)

Tokens of weight 0 (a prompt, padding) and those whose target is ``ignore_index`` are left out whatever their hidden states
hold, NaN among them: they add nothing to the loss, their log probability is given as 0, their gradient is 0, and the products
of more than 16 tokens are formed without their rows.  A target outside [0, V) of a token that counts makes the loss, that
token's gradient and the weight's NaN (it cannot be refused without waiting for the GPU).

The logits are formed in fp32 of exact products. For the gradients, softmax - onehot, times the token's weight over the largest
one, is rounded once to x's dtype as an operand of two more products, in pieces of the vocabulary (of up to 8 tokens whose
logits were kept it is not rounded); it is formed of the logits that the forward kept, where they take up to 2 GiB (and C is
768 or more, of float32 256, or the tokens are few), or of logits that are formed again. Of float32 operands the products are
those of linear_act; of many tokens the logits, and from kept logits the gradients, are formed of fp16 parts, which hold a
value to 2^-24 of itself and to 2^-40 of its row's largest (of the gradients' sums, of the largest term in their row of x or
column of the vocabulary). Beside copies of operands whose rows are no whole four-byte words, a call takes workspace in
proportion to the tokens (their rows of x, the sums of its gradient, eight bytes for each 32 to 256 columns) and up to some 0.5
GB for pieces of the vocabulary, whatever its size. Kept logits (float32, [T, V]) are held until the backward's graph is freed;
without gradients, or with ``keep_logits`` false, none are.

x and weight are taken as they are, under torch.autocast too; there, where their dtypes differ (a 16-bit hidden state and a
head's float32 weight), both are brought to the autocast dtype, as nn.Linear does, and gradients have the tensors' own.

``linear_cross_entropy`` is differentiable in x and weight (once); ``linear_cross_entropy_and_grad`` returns the gradients with
the loss, for a caller without autograd.
"""

from __future__ import annotations

import contextlib

import torch

from . import ops
from .int8 import call
from .linear import _autocast_dtype
from .policy import _check_denominator
from .profiling import timed

__all__ = ["linear_cross_entropy", "linear_cross_entropy_and_grad", "linear_cross_entropy_reference"]


def _check(denominator, ignore_index):
    return _check_denominator(denominator), int(ignore_index)


def _as_one(x, weight):
    """x and weight in one dtype, where autocast has one for them."""
    cast = _autocast_dtype(x) if x.dtype != weight.dtype else None
    if cast is None or torch.float64 in (x.dtype, weight.dtype) or not (x.is_floating_point() and weight.is_floating_point()):
        return x, weight
    return x.to(cast), weight.to(cast)


class LinearCrossEntropyFn(torch.autograd.Function):
    """linear_cross_entropy with its host steps in Python: under a kernel timer, and for torch.jit.trace, which records it."""

    @staticmethod
    def forward(ctx, x, weight, targets, mask, keep_logits, *numbers):
        with timed("linear_cross_entropy_fwd"):
            keep = keep_logits and any(ctx.needs_input_grad[:2])
            loss, logp, state = ops._binding().linear_ce_fwd(x, weight, targets, mask, *numbers, keep)
        ctx.save_for_backward(x, weight, targets, mask, state)
        ctx.numbers = numbers
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _dlogp):
        if dloss is None:
            return (None,) * 7
        *tensors, state = ctx.saved_tensors
        with timed("linear_cross_entropy_bwd"):
            dx, dw = ops._binding().linear_ce_bwd(*tensors, *ctx.numbers, state, dloss, *ctx.needs_input_grad[:2])
        return dx, dw, None, None, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None = None,
                         denominator: float | None = None, ignore_index: int = -100, keep_logits: bool = True):
    """(loss, logp): the scalar loss, differentiable in ``x`` and ``weight``, and each token's log probability (no gradient).

    x [..., C] and weight [V, C] float32, bfloat16 or float16, of one dtype; targets [...] int64 or int32; mask [...] bool
    or uint8 (a token counts where it is not 0), or floating weights.  With ``keep_logits`` false none are held for the
    backward, which then forms them again.
    """
    numbers = _check(denominator, ignore_index)
    x, weight = _as_one(x, weight)
    if ops._use_binding() and torch.autograd.forward_ad._current_level < 0:  # (forward mode is refused by the Function)
        return ops._binding().linear_ce(x, weight, targets, mask, *numbers, bool(keep_logits))
    return LinearCrossEntropyFn.apply(x, weight, targets, mask, bool(keep_logits), *numbers)


def linear_cross_entropy_and_grad(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None = None,
                                  denominator: float | None = None, ignore_index: int = -100, grad_scale: float = 1.0,
                                  keep_logits: bool = True):
    """(loss, logp, dx, dweight): linear_cross_entropy and grad_scale times its gradients, in the tensors' dtypes. No autograd.

    ``grad_scale`` is the loss scale of float16 training (the loss itself is not scaled); ``keep_logits`` as there.
    """
    numbers = _check(denominator, ignore_index)
    xs, ws = _as_one(x, weight)
    loss, logp, dx, dw = call("linear_ce_and_grad", xs, ws, targets, mask, *numbers, float(grad_scale), bool(keep_logits))
    return loss, logp, dx.to(x.dtype), dw.to(weight.dtype)


def linear_cross_entropy_reference(x, weight, targets, mask=None, denominator=None, ignore_index: int = -100):
    """linear_cross_entropy in elementary torch operations (fp32 for half inputs, else the inputs' dtype), on any device."""
    den, ignored = _check(denominator, ignore_index)
    up = torch.float64 if x.dtype == torch.float64 else torch.float32
    if mask is not None and mask.dtype == torch.uint8:
        mask = mask != 0
    w = torch.ones(targets.shape, dtype=up, device=x.device) if mask is None else mask.to(up)
    w = torch.where(targets == ignored, 0.0, w)
    live = w != 0
    with torch.autocast(x.device.type, enabled=False) if _autocast_dtype(x) else contextlib.nullcontext():
        z = torch.matmul(torch.where(live[..., None], x.to(up), 0.0), weight.to(up).t())
    at = torch.where(live, targets, 0).long()
    bad = (at < 0) | (at >= weight.shape[0])
    picked = z.gather(-1, torch.where(bad, 0, at)[..., None])[..., 0]
    logp = torch.where(bad, float("nan"), picked - torch.logsumexp(z, -1))
    logp = torch.where(live, logp, 0.0)
    total = den or w.sum()
    loss = -torch.where(live, w * logp, 0.0).sum() / (total if den else torch.where(total != 0, total, 1.0))
    return loss, logp.detach()
