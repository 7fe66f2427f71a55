"""The operators together: examples/policy_step.py learns, and a step through them is one through their plain forms."""

import importlib.util
from pathlib import Path

import pytest
import torch

from mhc_mlx_amd import policy_loss
from mhc_mlx_amd.linear import FusedLinear, linear_act_reference

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "policy_step.py"
    spec = importlib.util.spec_from_file_location("policy_step", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_example_learns():
    chances = _example().train(steps=12, say=lambda *_: None)
    assert chances[-1] > 20 * chances[0]


def test_gradients_through_the_model(monkeypatch):
    """float32 throughout: every parameter's gradient against the same model with plain products and torch's loss."""
    mod = _example()
    torch.manual_seed(1)
    model = mod.Policy(64, 32, 2, 4, dtype=torch.float32)
    state, actions = torch.randint(0, 64, (96,), device="cuda"), torch.randint(0, 64, (96,), device="cuda")
    adv = torch.randn(96, device="cuda")
    with torch.no_grad():
        old = mod.logp_of(model(state), actions) + 0.1 * torch.randn(96, device="cuda")
    policy_loss(model(state), actions, old, adv)[0].backward()
    got = {k: p.grad.clone() for k, p in model.named_parameters() if p.grad is not None}  # (MHCRewire has no RMSNorm)
    model.zero_grad()
    monkeypatch.setattr(FusedLinear, "forward", lambda self, x, residual=None: linear_act_reference(
        x, self.weight, self.bias, residual, self.activation, self.return_dtype))
    ratio = torch.exp(mod.logp_of(model(state), actions) - old)
    (-torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv).mean()).backward()
    assert len(got) > 10
    for k, p in model.named_parameters():
        if k not in got:
            continue
        # a few hundred fp32 roundings of values of the gradient's size on either side
        assert (got[k] - p.grad).abs().max() <= 2e-5 * p.grad.abs().max() + 1e-9, k
