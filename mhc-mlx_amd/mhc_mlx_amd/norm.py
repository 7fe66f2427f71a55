"""add_rms_norm: RMS norm with the residual's addition, AddRMSNorm, the module over it, and its int8 form for serving.

    h = x + residual, rounded to their dtype
    y = h / sqrt(mean(h^2) + eps) * weight

It closes a block beside ``residual_add_agg``: h goes on as the residual stream, y into the next product.  x and residual
are [..., C] of one dtype (float32, bfloat16 or float16), weight [C] of that dtype or float32; what is normed is h as it is
stored.  Sums are held in fp32 (squares past its range are summed scaled).  The backward gives the gradients of x (which are
the residual's too) and of the weight, from those of y and h.  It is not twice differentiable.

``add_rms_norm_int8`` gives y as ``Int8Rows``: int8 codes and a float32 scale for each row (its largest magnitude over 127),
as ``linear_int8`` takes them.  A row of zeros has the scale 0, one with an infinity or NaN the scale NaN.  No autograd.

The functions need GPU tensors and the built library; AddRMSNorm hands a call that the HIP path cannot take (CPU tensors, a
RuntimeError from the library) to ``add_rms_norm_reference``, with one warning per process, as MHCLayer does.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import layer, ops
from .int8 import Int8Rows, call, quantize_int8_reference
from .profiling import timed

__all__ = ["AddRMSNorm", "add_rms_norm", "add_rms_norm_int8", "add_rms_norm_reference"]


def _check_eps(eps) -> float:
    # (as the kernels take it: a float32)
    if not 2.0 ** -126 <= eps < math.inf:
        raise ValueError(f"eps must be positive (at least 2^-126) and finite (got {eps})")
    return float(eps)


class AddRMSNormFn(torch.autograd.Function):
    """add_rms_norm with its host steps in Python: under a kernel timer, and for torch.jit.trace, which records it."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        with timed("add_rms_norm_fwd"):
            y, h, rstd = ops._binding().add_rms_norm_fwd(x, residual, weight, eps, True)
        ctx.save_for_backward(x if h is None else h, rstd, weight)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        if dy is None and dh is None:
            return (None,) * 4
        h, rstd, weight = ctx.saved_tensors
        of_x, of_r, of_w, _ = ctx.needs_input_grad
        with timed("add_rms_norm_bwd"):
            dx, dw = ops._binding().add_rms_norm_bwd(dy, dh, h, rstd, weight, of_x or of_r, of_w)
        return dx if of_x else None, dx if of_r else None, dw, None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(y, h): the normed sum and the sum itself (x without a residual), differentiable in all three tensors.

    Rows of x and residual may lie any distance apart; other strides are copied.
    """
    eps = _check_eps(eps)
    if ops._use_binding() and torch.autograd.forward_ad._current_level < 0:  # (forward mode is refused by the Function)
        y, h = ops._binding().add_rms_norm(x, residual, weight, eps)
        return y, x if residual is None else h
    out = AddRMSNormFn.apply(x, residual, weight, eps)
    return (out, x) if residual is None else out


def add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(Int8Rows of y, h): add_rms_norm with its output in 8 bits. No autograd."""
    eps = _check_eps(eps)
    if ops._use_binding():
        codes, scales, h = ops._binding().add_rms_norm_int8(x, residual, weight, eps)
    else:
        codes, scales, h = call("add_rms_norm_int8", x, residual, weight, eps)
    return Int8Rows(codes, scales), x.detach() if residual is None else h


def add_rms_norm_reference(x, residual=None, weight=None, eps: float = 1e-6, int8: bool = False):
    """add_rms_norm (or with ``int8`` its int8 form) in elementary torch operations (fp32 for half inputs), on any device."""
    eps = _check_eps(eps)
    up = torch.float64 if x.dtype == torch.float64 else torch.float32
    h = x if residual is None else (x.to(up) + residual.to(up)).to(x.dtype)
    z = h.to(up)
    y = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(up)
    return (quantize_int8_reference(y) if int8 else y.to(x.dtype)), h


class AddRMSNorm(nn.Module):
    """add_rms_norm with a weight of its own (ones at the start; ``dtype`` may be the rows' or float32).

    ``forward(x, residual=None)`` gives (y, h); with ``int8`` y is Int8Rows, without autograd, for an Int8Linear behind it.
    x and a residual of different dtypes (one of them from an autocast region) are brought to the one that their sum has,
    and a weight of neither that dtype nor float32 to float32.
    """

    def __init__(self, dim: int, eps: float = 1e-6, *, int8: bool = False, device=None, dtype=None):
        super().__init__()
        self.dim, self.eps, self.int8 = int(dim), _check_eps(eps), bool(int8)
        self.weight = nn.Parameter(torch.ones(self.dim, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if residual is not None and residual.dtype != x.dtype:
            both = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(both), residual.to(both)
        weight = self.weight if self.weight.dtype in (x.dtype, torch.float32) else self.weight.float()
        if not layer._disabled_by_env() and layer.hip_available():
            why = layer._off_gpu(x, residual, self.weight)
            if why is None:
                try:
                    return (add_rms_norm_int8 if self.int8 else add_rms_norm)(x, residual, weight, self.eps)
                except RuntimeError as e:
                    why = e
            layer._fallback_warning(" in AddRMSNorm", why)
        if self.int8:
            with torch.no_grad():
                return add_rms_norm_reference(x, residual, weight, self.eps, int8=True)
        return add_rms_norm_reference(x, residual, weight, self.eps)

    def extra_repr(self) -> str:
        return f"{self.dim}, eps={self.eps}" + (", int8=True" if self.int8 else "")
