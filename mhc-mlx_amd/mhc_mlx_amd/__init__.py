"""mhc_mlx_amd — the fused mHC layer of svdrecbd/mhc-mlx on MI355X (gfx950).

``MHCLayer`` / ``MHCRewire`` keep the reference's module API; the hot path
runs in libmhc_hip.so (hand-written HIP kernels, C ABI in include/mhc_hip.h).
``FusedLinear`` / ``linear_act``, ``policy_loss`` and ``AdamW`` are the rest of
a training step around it: the layer it connects, a loss and the update.
``AddRMSNorm`` / ``add_rms_norm``, ``Int8Linear`` / ``linear_int8`` and
``linear_cross_entropy`` lie between the residual stream and a model's answer.
"""

from . import tuning

tuning.load()  # the tuning files of the working directory and ~/.cache/mhc-mlx (metal.py:21-33)

from .layer import MHCLayer, MHCRewire  # noqa: E402
from .patching import AutoPatcher  # noqa: E402
from . import ops, reference  # noqa: E402
from .ops import (  # noqa: E402
    mhc_forward_fused_hip,
    mhc_forward_fused_hip_autograd,
    mhc_layer_forward,
    mhc_layer_forward_dynamic,
    post_combine,
    residual_add_agg_hip,
    sinkhorn_knopp_hip,
    sinkhorn_knopp_hip_autograd,
    stream_mix_add_hip,
    stream_mix_add_hip_autograd,
    stream_scale,
)
from .cross_entropy import linear_cross_entropy, linear_cross_entropy_and_grad  # noqa: E402
from .int8 import Int8Linear, Int8Rows, linear_int8, quantize_int8  # noqa: E402
from .linear import FusedLinear, linear_act  # noqa: E402
from .norm import AddRMSNorm, add_rms_norm, add_rms_norm_int8  # noqa: E402
from .optim import AdamW, adamw_step_hip  # noqa: E402
from .policy import policy_loss, policy_loss_and_grad  # noqa: E402
from .profiling import kernel_timer  # noqa: E402
from .utils import residual_add_agg  # noqa: E402

__version__ = "0.1.0"

__all__ = [
    "AdamW",
    "AddRMSNorm",
    "AutoPatcher",
    "FusedLinear",
    "Int8Linear",
    "Int8Rows",
    "MHCLayer",
    "MHCRewire",
    "ops",
    "reference",
    "adamw_step_hip",
    "add_rms_norm",
    "add_rms_norm_int8",
    "kernel_timer",
    "linear_act",
    "linear_cross_entropy",
    "linear_cross_entropy_and_grad",
    "linear_int8",
    "mhc_forward_fused_hip",
    "mhc_forward_fused_hip_autograd",
    "mhc_layer_forward",
    "mhc_layer_forward_dynamic",
    "policy_loss",
    "policy_loss_and_grad",
    "post_combine",
    "quantize_int8",
    "residual_add_agg",
    "residual_add_agg_hip",
    "sinkhorn_knopp_hip",
    "sinkhorn_knopp_hip_autograd",
    "stream_mix_add_hip",
    "stream_mix_add_hip_autograd",
    "stream_scale",
    "__version__",
]
