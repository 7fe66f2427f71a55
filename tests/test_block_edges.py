"""The cross entropy's and the policy loss's numbers and masks at their ends, without a GPU."""

import math

import pytest
import torch

from mhc_mlx_amd import linear_cross_entropy, linear_cross_entropy_and_grad, policy_loss, policy_loss_and_grad
from mhc_mlx_amd.cross_entropy import linear_cross_entropy_reference


@pytest.mark.parametrize("bad", [1e-50, 1e-40, 2.0 ** -127, 1e39, math.inf, math.nan])
def test_denominators_that_are_no_float32_are_refused(bad):
    """1e-50 is 0 there, and 0 asks for the sum of the weights."""
    x, y, t = torch.zeros(2, 4), torch.zeros(2, dtype=torch.long), torch.zeros(2)
    for call in (linear_cross_entropy, linear_cross_entropy_and_grad):
        with pytest.raises(ValueError, match="denominator"):
            call(x, x, y, denominator=bad)
    for call in (policy_loss, policy_loss_and_grad):
        with pytest.raises(ValueError, match="denominator"):
            call(x, y, t, t, denominator=bad)


def test_denominators_that_are_taken():
    x, y, t = torch.zeros(2, 4), torch.zeros(2, dtype=torch.long), torch.zeros(2)
    for good in (2.0 ** -126, 3, torch.finfo(torch.float32).max):
        for call in (lambda: linear_cross_entropy(x, x, y, denominator=good), lambda: policy_loss(x, y, t, t, denominator=good)):
            with pytest.raises(ValueError, match="GPU"):  # (the next check)
                call()


def test_byte_masks_of_the_plain_form():
    """A byte other than 0 is 1, as in the kernels."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(6, 5, generator=g), torch.randn(7, 5, generator=g)
    y, mask = torch.arange(6), torch.tensor([1, 3, 0, 255, 2, 0], dtype=torch.uint8)
    want = linear_cross_entropy_reference(x, w, y, mask != 0)
    got = linear_cross_entropy_reference(x, w, y, mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_plain_form_under_autocast():
    """Its logits stay in float32."""
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 50, generator=g), torch.randn(7, 50, generator=g)
    want = linear_cross_entropy_reference(x, w, torch.arange(6))
    with torch.autocast("cpu", torch.bfloat16):
        got = linear_cross_entropy_reference(x, w, torch.arange(6))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
