"""AdamW over many tensors at once, with states in 32 or in 8 bits.

A model with mHC layers has many small parameters (n, n, n * n and C floats for every layer) next to large ones.  One
step updates them all in a few launches, each of which takes as many tensors of any size as its kernel arguments hold
addresses of: 100 with 32-bit states, 84 with masters or 8-bit states, 72 with both.

    p <- p (1 - lr weight_decay);  m <- b1 m + (1 - b1) g;  v <- b2 v + (1 - b2) g g
    p <- p - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)

in fp32, every operation rounded by itself, so that results do not depend on how the tensors are split up.  A 16-bit
parameter may have a float32 master copy that is updated in its place (the parameter is its rounding).

States in 8 bits are e4m3 codes of m and of sqrt(v), in blocks of 256 elements with a float32 unit each: the largest
value of a block is 448 units, values below 2^-10 units are 0, and a code is within 1/16 of its value above 2^-6 units.
(v is kept as its root since a code spans 2^18: enough for sqrt(v), not for v.)  A non-finite gradient costs its whole
block the state.

``adamw_step_hip`` is one step over lists of tensors; ``AdamW`` is the torch optimizer over it.
"""

from __future__ import annotations

import itertools
import math

import torch

from . import layer, ops
from .profiling import timed

__all__ = ["AdamW", "adamw_step_hip", "adamw_step_reference"]

BLOCK = 256  # elements of an 8-bit state that share a unit
_CODE_MAX = 448.0
_MIN_TOP = 2.0 ** -100


def _check_numbers(step, lr, betas, eps, weight_decay) -> None:
    if not (lr >= 0 and eps >= 0 and weight_decay >= 0):
        raise ValueError(f"lr, eps and weight_decay must be >= 0 (got {lr}, {eps}, {weight_decay})")
    if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
        raise ValueError(f"betas must be two numbers in [0, 1) (got {betas})")
    if isinstance(step, bool) or not isinstance(step, int) or step < 1:
        raise ValueError(f"step must be an integer >= 1 (got {step!r})")


def adamw_step_hip(params, grads, exp_avgs, exp_avg_sqs, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                   weight_decay: float = 0.01, masters=None, scales=None, grad_scale=1.0) -> None:
    """One AdamW step over lists of tensors, in place. No autograd.

    params and grads: float32, bfloat16 or float16, a gradient of its parameter's dtype and shape (one of another layout
    is copied).  exp_avgs, exp_avg_sqs: float32, or, with ``scales``, float8_e4m3fn codes of m and sqrt(v); a scales
    entry is float32 [ceil(numel / 256), 2], the units of both in each block of 256 elements in memory order.  masters:
    None, or a float32 copy or None for each parameter.  States and masters have their parameter's layout.  ``step`` counts from
    1.  ``grad_scale`` multiplies the gradients: a number, or one float32 on the GPU (a clipping factor, without waiting for it).
    The call only enqueues work; a captured graph replays it with the step's numbers as they were.
    """
    _check_numbers(step, lr, betas, eps, weight_decay)
    scale_t = grad_scale if isinstance(grad_scale, torch.Tensor) else None
    with timed("adamw_step"):
        ops._binding().adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, scales, step, float(lr), float(betas[0]),
                                  float(betas[1]), float(eps), float(weight_decay), 1.0 if scale_t is not None else float(grad_scale),
                                  scale_t)


def _decode(codes: torch.Tensor, units: torch.Tensor) -> torch.Tensor:
    return codes.float() * units.repeat_interleave(BLOCK)[:codes.numel()]


def _encode(t: torch.Tensor):
    blocks = torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)
    top = blocks.abs().amax(1).clamp(min=_MIN_TOP)
    return (blocks * (top.reciprocal() * _CODE_MAX)[:, None]).view(-1)[:t.numel()].to(torch.float8_e4m3fn), top * (1.0 / _CODE_MAX)


def _in_memory_order(t: torch.Tensor) -> torch.Tensor:
    """t's elements as they lie in memory (t has no holes): 1-d, sharing its storage."""
    return t.as_strided((t.numel(),), (1,))


@torch.no_grad()
def adamw_step_reference(params, grads, exp_avgs, exp_avg_sqs, step: int, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                         weight_decay: float = 0.01, masters=None, scales=None, grad_scale=1.0) -> None:
    """adamw_step_hip in elementary torch operations, on any device: the same roundings, so the same results."""
    _check_numbers(step, lr, betas, eps, weight_decay)
    b1, b2 = betas
    for i, p in enumerate(params):
        if p.numel() == 0:
            continue
        flat = _in_memory_order(p)
        w = flat if masters is None or masters[i] is None else _in_memory_order(masters[i])
        g = _in_memory_order(torch.empty_like(p, dtype=torch.float32).copy_(grads[i])) * grad_scale
        m, v = _in_memory_order(exp_avgs[i]), _in_memory_order(exp_avg_sqs[i])
        m32, v32 = (m, v) if scales is None else (_decode(m, scales[i][:, 0]), _decode(v, scales[i][:, 1]).square())
        new = w.float() * (1.0 - lr * weight_decay)
        m32 = m32 * b1 + g * (1.0 - b1)
        v32 = v32 * b2 + (g * g) * (1.0 - b2)
        root = torch.sqrt(v32.double()).float()  # (torch's fp32 square root on the CPU is not always the nearest)
        new = new - (m32 / (root * (1.0 / math.sqrt(1.0 - b2 ** step)) + eps)) * (lr / (1.0 - b1 ** step))
        if scales is not None:
            m32, mu = _encode(m32)
            v32, vu = _encode(root)
            scales[i].copy_(torch.stack([mu, vu], 1))
        for t, value in ((m, m32), (v, v32), (flat, new)) + (((w, new),) if w is not flat else ()):
            t.copy_(value)


class AdamW(torch.optim.Optimizer):
    """torch optimizer over adamw_step_hip.

    ``state_bits`` 8 keeps the states of tensors with at least ``min_8bit_size`` elements in 8 bits (those of smaller ones,
    the mHC parameters among them, in 32).  ``master_weights`` gives every 16-bit parameter a float32 master copy, made from
    it at its first step; the parameter is the copy's rounding from then on, so that one who sets a parameter's values
    later sets ``state[p]["master"]`` too.  CPU parameters are updated by ``adamw_step_reference``.  ``step(grad_scale=...)`` multiplies
    the gradients.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *,
                 state_bits: int = 32, min_8bit_size: int = 4096, master_weights: bool = True):
        _check_numbers(1, lr, betas, eps, weight_decay)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32 (got {state_bits})")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=min_8bit_size, master_weights=master_weights))

    @staticmethod
    def _new_state(p: torch.Tensor, group: dict) -> dict:
        s = {"step": 0}
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            # float8 zeros are the byte 0
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
            s["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
            s["scales"] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, 2, dtype=torch.float32, device=p.device)
        else:
            s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            s["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        if group["master_weights"] and p.dtype in (torch.float16, torch.bfloat16):
            s["master"] = p.detach().clone().float()
        return s

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale=1.0):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls: dict = {}  # tensors that one call can take: of one device, step and width of states
            for p in group["params"]:
                if p.grad is None:
                    continue
                s = self.state[p]
                if not s:
                    s.update(self._new_state(p, group))
                s["step"] += 1
                calls.setdefault((p.device, s["step"], "scales" in s), []).append((p, s))
            for (device, step, coded), tensors in calls.items():
                states = [s for _, s in tensors]
                hip = device.type == "cuda" and not layer._disabled_by_env()
                (adamw_step_hip if hip else adamw_step_reference)(
                    [p for p, _ in tensors], [p.grad for p, _ in tensors], [s["exp_avg"] for s in states],
                    [s["exp_avg_sq"] for s in states], step, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                    masters=[s.get("master") for s in states], scales=[s["scales"] for s in states] if coded else None,
                    grad_scale=grad_scale)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but states keep the dtypes they were saved with (torch casts them to their parameter's)."""
        super().load_state_dict(state_dict)
        saved = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        mine = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for key, p in zip(saved, mine):
            for name, value in state_dict["state"].get(key, {}).items():
                if isinstance(value, torch.Tensor):
                    self.state[p][name] = value.detach().clone().to(p.device)
