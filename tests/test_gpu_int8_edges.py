"""linear_int8: residuals whose ends are no whole words."""

import pytest
import torch

from mhc_mlx_amd import Int8Rows, linear_int8
from tests._block import int8_product64
from tests._train import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(129, 255, 64), (401, 1023, 256), (1001, 2049, 1100), (2049, 4097, 128)])
def test_residuals_that_start_and_end_anywhere(M, N, K, dt):
    """Of an odd number of elements, from an odd one on, with nothing behind the last."""
    g = torch.Generator(device="cuda").manual_seed(M)
    codes = lambda n: torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    x, w = Int8Rows(codes(M), torch.rand(M, generator=g, device="cuda") * 0.02), Int8Rows(codes(N), torch.rand(N, generator=g, device="cuda") * 0.02)
    held = torch.randn(M * N + 1, generator=g, device="cuda").to(dt)
    r = held[1:].view(M, N)
    out = linear_int8(x, w, None, r, "silu", dt)
    close(out, *int8_product64(x, w, None, r, "silu", dt))
    assert torch.equal(out, linear_int8(x, w, None, r.clone(), "silu", dt))
