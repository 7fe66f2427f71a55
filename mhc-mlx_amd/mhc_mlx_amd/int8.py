"""linear_int8: a product of int8 rows with scales for each token and channel, and Int8Linear, the module over it.

    out = act(x.scales weight.scales (x.codes weight.codes^T) + bias) + residual

``Int8Rows`` holds codes (int8, [..., K]) and scales (float32, [...]): a row's values are its codes times its scale.
``quantize_int8`` makes them of float32, bfloat16 or float16 rows (codes are rint(127 x / max|x|)), ``add_rms_norm_int8`` of
normed ones.  The products' sums are exact (32-bit whole numbers, K below 2^17), or those of up to 16 parts of them where there
are few outputs, and are scaled and added up in fp32 (times x's scale they have to stay in its range); the output is float32,
bfloat16 or float16, the residual of its dtype, the bias of any floating dtype (read as float32).

All of it is for serving: nothing here has a gradient, and results of inputs that require one carry none.

The functions need GPU tensors and the built library; Int8Linear hands a call that the HIP path cannot take (CPU tensors, a
wider layer, a RuntimeError from the library) to ``linear_int8_reference``, with one warning per process, as MHCLayer does.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from . import layer, ops
from .linear import _act_code, linear_act_reference
from .profiling import timed

__all__ = ["Int8Linear", "Int8Rows", "linear_int8", "linear_int8_reference", "quantize_int8", "quantize_int8_reference"]

_MAX_K, _MAX_N = 1 << 17, 1 << 22  # K and N stay below them


class Int8Rows(NamedTuple):
    """Rows in 8 bits: ``codes`` (int8, [..., K]) times ``scales`` (float32, [...])."""

    codes: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the rows stand for."""
        if self.codes.is_cuda and dtype != torch.float64:
            return call("dequantize_int8", self.codes, self.scales, ops._code(dtype))
        out = torch.empty(self.codes.shape, dtype=dtype, device=self.codes.device)
        return torch.mul(self.codes, self.scales.unsqueeze(-1), out=out)


class RecordedFn(torch.autograd.Function):
    """A call of the binding without a gradient, as a node that torch.jit.trace keeps and runs again."""

    @staticmethod
    def forward(ctx, name, *args):
        out = getattr(ops._binding(), name)(*args)
        ctx.mark_non_differentiable(*(out if isinstance(out, tuple) else (out,)))
        return out

    @staticmethod
    def backward(ctx, *grads):  # pragma: no cover - its results are not differentiable
        return None


def call(name: str, *args):
    """A call of the binding without a gradient, under a kernel timer or while torch.jit.trace records."""
    if torch._C._is_tracing():
        return RecordedFn.apply(name, *args)
    with timed(name):
        return getattr(ops._binding(), name)(*args)


def quantize_int8(x: torch.Tensor) -> Int8Rows:
    """x [..., K] in 8 bits, with a scale for each row. Rows may lie any distance apart; other strides are copied."""
    if ops._use_binding():
        return Int8Rows(*ops._binding().quantize_int8(x))
    return Int8Rows(*call("quantize_int8", x))


def linear_int8(x: Int8Rows, weight: Int8Rows, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                activation: str = "none", output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """act(x weight^T + bias) + residual of rows in 8 bits: x [..., K], weight [N, K], bias [N], residual [..., N].

    ``activation`` is one of ``linear.ACTIVATIONS``.  Rows of codes may lie any distance apart; those that are no whole
    four-byte words (an odd K) are copied in every call.
    """
    act, out_code = _act_code(activation), ops._code(output_dtype)
    if ops._use_binding():
        return ops._binding().linear_int8(x[0], x[1], weight[0], weight[1], bias, residual, act, out_code)
    return call("linear_int8", x[0], x[1], weight[0], weight[1], bias, residual, act, out_code)


@torch.no_grad()
def quantize_int8_reference(x: torch.Tensor) -> Int8Rows:
    """quantize_int8 in elementary torch operations (in float64: halves have to be seen as such), on any device."""
    z = x.double()
    top = z.abs().amax(-1, keepdim=True)
    good = torch.isfinite(top)
    codes = torch.round(127.0 * z / torch.where(good & (top > 0), top, 1.0))
    scales = torch.where(good, top, float("nan")) / 127.0
    return Int8Rows(torch.where(good, codes, 0.0).to(torch.int8), scales.squeeze(-1).float())


@torch.no_grad()
def linear_int8_reference(x, weight, bias=None, residual=None, activation: str = "none", output_dtype=torch.bfloat16):
    """linear_int8 in elementary torch operations (the sums in float64, where they are exact), on any device."""
    sums = torch.matmul(x[0].double(), weight[0].double().t()).float() * x[1].unsqueeze(-1) * weight[1]
    # (a product with the unit matrix of one column hands the sums to the plain epilogue as they are)
    z = sums if bias is None else sums + bias.float()
    one = torch.ones(1, 1, device=z.device)
    out = linear_act_reference(z.reshape(-1, 1), one, None, None, activation).reshape(z.shape)
    return (out if residual is None else out + residual.float()).to(output_dtype)


class Int8Linear(nn.Module):
    """A Linear in 8 bits: int8 weights with a scale for each output, and activations in 8 bits with one for each token.

    ``forward(x, residual=None)`` takes a floating x, which it quantizes, or Int8Rows.  The output has ``return_dtype``, or
    x's dtype (float32 for Int8Rows).  ``from_linear`` makes one of an nn.Linear or FusedLinear.  Weights, scales and bias
    are buffers (the latter two float32 whatever the module is cast to); AutoPatcher wraps it as a quantized Linear.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str = "none", *,
                 return_dtype: torch.dtype | None = None, device=None):
        _act_code(activation)
        if return_dtype is not None:
            ops._code(return_dtype)
        super().__init__()
        self.in_features, self.out_features = int(in_features), int(out_features)
        self.activation, self.return_dtype = activation, return_dtype
        self.register_buffer("weight", torch.zeros(self.out_features, self.in_features, dtype=torch.int8, device=device))
        self.register_buffer("weight_scale", torch.zeros(self.out_features, device=device))
        self.register_buffer("bias", torch.zeros(self.out_features, device=device) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "Int8Linear":
        """The layer's weights in 8 bits; a FusedLinear's activation is kept, and the output's dtype is the layer's."""
        weight = linear.weight.detach()
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, getattr(linear, "activation", "none"),
                return_dtype=getattr(linear, "return_dtype", None) or weight.dtype, device=weight.device)
        rows = quantize_int8(weight) if weight.is_cuda and not layer._disabled_by_env() else quantize_int8_reference(weight)
        m.weight.copy_(rows.codes)
        m.weight_scale.copy_(rows.scales)
        if linear.bias is not None:
            m.bias.copy_(linear.bias)
        return m

    def _apply(self, fn, recurse=True):
        held = {k: getattr(self, k) for k in ("weight_scale", "bias")}
        super()._apply(fn, recurse)
        for k, t in held.items():  # a cast of the module is not one of its scales
            if t is not None and getattr(self, k).dtype != torch.float32:
                setattr(self, k, t.to(self.weight.device))
        return self

    def forward(self, x: torch.Tensor | Int8Rows, residual: torch.Tensor | None = None) -> torch.Tensor:
        given = isinstance(x, tuple)
        weight = Int8Rows(self.weight, self.weight_scale)
        dtype = self.return_dtype or (torch.float32 if given else x.dtype)
        if not layer._disabled_by_env() and layer.hip_available():
            why = layer._off_gpu(*(x if given else (x,)), self.weight, residual)
            if self.in_features >= _MAX_K or self.out_features >= _MAX_N:
                why = f"the HIP path needs in_features below {_MAX_K} and out_features below {_MAX_N}"
            if why is None:
                try:
                    return linear_int8(x if given else quantize_int8(x), weight, self.bias, residual, self.activation, dtype)
                except RuntimeError as e:
                    why = e
            layer._fallback_warning(" in Int8Linear", why)
        return linear_int8_reference(x if given else quantize_int8_reference(x), weight, self.bias, residual, self.activation, dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, activation={self.activation}"
