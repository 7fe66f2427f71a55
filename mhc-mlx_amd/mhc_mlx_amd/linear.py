"""linear_act: a matrix product with bias, activation and residual in its epilogue, and FusedLinear, the module over it.

    out = act(x W^T + bias) + residual

It is the layer that MHCRewire wraps and AutoPatcher finds (FusedLinear is an ``nn.Linear``).  x is [..., K], weight
[N, K], bias [N], residual [..., N]; float32, bfloat16 or float16, x, weight and bias of one dtype; the output (and the
residual) of that dtype or float32.  Sums are held in fp32.  The backward gives the gradients of x, weight, bias and
residual; dz = dout act'(z) is rounded once to x's dtype as an operand of the two products (the bias's gradient is
summed from it unrounded).  The forward keeps act'(z) for it, of 16-bit operands in 16 bits (to 2^-16, and to 2^-10 of
itself down to 2^-29), and forms their activations to about 2^-21 of z and 2^-15 of themselves, for float32 outputs too.
It is not twice differentiable.

linear_act needs GPU tensors and the built library, fewer than 2^28 rows, and N and K below 2^22; FusedLinear hands a call
that the HIP path cannot take (CPU tensors, a wider layer, a RuntimeError from the library) to ``linear_act_reference``,
with one warning per process, as MHCLayer does.

Under torch.autocast FusedLinear casts x, weight and bias to the autocast dtype, as nn.Linear does; linear_act takes its
arguments as they are.
"""

from __future__ import annotations

import contextlib
import math

import torch
import torch.nn as nn

from . import _lib, layer, ops
from .profiling import timed

__all__ = ["ACTIVATIONS", "FusedLinear", "linear_act", "linear_act_reference"]

ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH,
               "silu": _lib.ACT_SILU}


_MAX_WIDTH = 1 << 22  # N and K stay below it


def _act_code(activation: str) -> int:
    try:
        return ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"activation must be one of: {', '.join(ACTIVATIONS)} (got {activation!r})") from None


def _autocast_dtype(x: torch.Tensor) -> torch.dtype | None:
    device = x.device.type
    return torch.get_autocast_dtype(device) if device in ("cuda", "cpu") and torch.is_autocast_enabled(device) else None


class LinearActFn(torch.autograd.Function):
    """linear_act with its host steps in Python: under a kernel timer, and for torch.jit.trace, which records it."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_code):
        want = any(ctx.needs_input_grad[:3])
        with timed("linear_act_fwd"):
            out, dact = ops._binding().linear_fwd(x, weight, bias, residual, act, out_code, want)
        ctx.save_for_backward(x, weight, dact)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        if dout is None:
            return (None,) * 6
        x, weight, dact = ctx.saved_tensors
        with timed("linear_act_bwd"):
            dx, dw, db = ops._binding().linear_bwd(dout, dact, x, weight, *ctx.needs_input_grad[:3])
        return dx, dw, db, dout if ctx.needs_input_grad[3] else None, None, None


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, activation: str = "none",
               output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, differentiable in all four tensors.

    ``activation`` is one of ``ACTIVATIONS`` (gelu is the one with the error function).  The output has x's dtype unless
    ``output_dtype`` is float32.  Rows of x and weight may lie any distance apart; other strides are copied.
    """
    act = _act_code(activation)
    out_code = ops._code(x.dtype if output_dtype is None else output_dtype)
    if ops._use_binding() and torch.autograd.forward_ad._current_level < 0:  # (forward mode is refused by the Function)
        return ops._binding().linear_act(x, weight, bias, residual, act, out_code)
    return LinearActFn.apply(x, weight, bias, residual, act, out_code)


def linear_act_reference(x, weight, bias=None, residual=None, activation: str = "none", output_dtype=None):
    """linear_act in elementary torch operations (fp32 for half inputs, else the inputs' dtype), on any device."""
    _act_code(activation)
    up = torch.float64 if x.dtype == torch.float64 else torch.float32
    with torch.autocast(x.device.type, enabled=False) if _autocast_dtype(x) else contextlib.nullcontext():
        z = torch.matmul(x.to(up), weight.to(up).t())
    if bias is not None:
        z = z + bias.to(up)
    if activation == "relu":
        z = torch.clamp(z, min=0.0)
    elif activation == "gelu":
        z = z * (0.5 * torch.erfc(z * -math.sqrt(0.5)))
    elif activation == "gelu_tanh":
        z = 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    elif activation == "silu":
        z = z * torch.sigmoid(z)
    if residual is not None:
        z = z + residual.to(up)
    return z.to(x.dtype if output_dtype is None else output_dtype)


class FusedLinear(nn.Linear):
    """nn.Linear with an activation, and an optional residual of its output's shape, in the product's epilogue.

    ``return_dtype`` (torch.float32, or None for x's dtype) is the output's dtype.  Parameters, their names and their
    initialisation are nn.Linear's, so checkpoints carry over and AutoPatcher wraps it like one.  Under autocast x's dtype
    is the autocast one, and a float32 residual makes the output float32, as adding it would.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", *,
                 return_dtype: torch.dtype | None = None, device=None, dtype=None):
        _act_code(activation)
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.activation = activation
        self.return_dtype = return_dtype

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        weight, bias, return_dtype = self.weight, self.bias, self.return_dtype
        cast = _autocast_dtype(x)
        if cast is not None and x.dtype != torch.float64:  # (autocast leaves float64 alone)
            x, weight, bias = x.to(cast), weight.to(cast), None if bias is None else bias.to(cast)
            if residual is not None:
                return_dtype = return_dtype or (torch.float32 if residual.dtype == torch.float32 else cast)
                residual = residual.to(return_dtype)
        if not layer._disabled_by_env() and layer.hip_available():
            why = layer._off_gpu(x, weight, bias, residual)
            if max(self.in_features, self.out_features) >= _MAX_WIDTH:
                why = f"the HIP path needs N and K below {_MAX_WIDTH} (got {self.out_features} and {self.in_features})"
            if why is None:
                try:
                    return linear_act(x, weight, bias, residual, self.activation, return_dtype)
                except RuntimeError as e:
                    why = e
            layer._fallback_warning(" in FusedLinear", why)
        return linear_act_reference(x, weight, bias, residual, self.activation, return_dtype)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
