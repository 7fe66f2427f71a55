"""linear_act / FusedLinear at the ends of what they take: very long rows, many rows, tiny values, mixed types."""

import pytest
import torch

from tests._train import close, linear64, linear_grads64

from mhc_mlx_amd import FusedLinear, linear_act
from mhc_mlx_amd import layer as L

pytestmark = pytest.mark.gpu


def test_rows_of_more_than_8_megabytes():
    """fp32 reductions past 2^21 elements, forward and in dx, at sizes that large tiles would serve best.

    The values are positive, so that a sum that lacks a part of its terms is far outside the bound.
    """
    M, N, K = 1024, 1024, 2_200_000
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = (torch.rand(n, K, generator=g, device="cuda") for n in (M, N))
    rows = torch.tensor([0, 127, 128, 190, 255, 256, 447, 1023], device="cuda")  # first, middle and last ones of tiles
    out = linear_act(x, w)
    ref, bound, *_ = linear64(x[rows], w[rows], None, None, "none", torch.float32)
    close(out[rows][:, rows], ref, bound, "out")
    del out
    # dx [1024, 1024] = dout [1024, K] W [K, 1024]
    wide = w.view(K, N)
    a = torch.rand(M, N, generator=g, device="cuda").requires_grad_(True)
    dx, = torch.autograd.grad(linear_act(a, wide), a, x)
    del w
    some = wide[:, rows]
    ones = torch.ones(len(rows), K, dtype=torch.float64, device="cuda")
    (ref, bound), _, _ = linear_grads64(a[rows][:, rows], some, x[rows], ones, torch.zeros_like(ones), torch.float32, False)
    close(dx[rows][:, rows], ref, bound, "dx")


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_more_than_2_22_rows(dt):
    """Zeros and ones, so that every sum over the rows is a whole number below 2^24: exact in fp32."""
    M, N, K = (1 << 22) + 70, 24, 16
    g = torch.Generator(device="cuda").manual_seed(6)
    x, w, up = (torch.randint(0, 2, s, generator=g, device="cuda").to(dt) for s in ((M, K), (N, K), (M, N)))
    b = torch.ones(N, device="cuda", dtype=dt)
    ts = [t.requires_grad_(True) for t in (x, w, b)]
    out = linear_act(*ts, activation="relu")
    xd, wd, ud = (t.detach().double() for t in (x, w, up))
    assert torch.equal(out, (xd @ wd.t() + 1).to(dt))
    dx, dw, db = torch.autograd.grad(out, ts, up)  # (every sum is positive: relu's derivative is 1)
    assert torch.equal(dx, (ud @ wd).to(dt)) and torch.equal(dw, (ud.t() @ xd).to(dt))
    assert torch.equal(db, (torch.ones(1, M, dtype=torch.float64, device="cuda") @ ud)[0].to(dt))


def test_wider_layers_than_the_kernels_take(monkeypatch):
    """linear_act refuses them, FusedLinear computes them in the plain form."""
    monkeypatch.setattr(L, "_METAL_FAILED", True)  # (the warning has been given)
    for N, K in ((2, 1 << 22), (1 << 22, 2)):
        m = FusedLinear(K, N, device="cuda")
        x = torch.randn(3, K, device="cuda")
        with pytest.raises(ValueError, match="2\\^22"):
            linear_act(x, m.weight, m.bias)
        ref, bound, *_ = linear64(x, m.weight, m.bias, None, "none", torch.float32)
        close(m(x), ref, bound, "out")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("given", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [5, 200])
def test_fused_linear_under_autocast(dt, given, rows):
    """The call and its gradients are those of the operands in the autocast dtype; parameters get float32 gradients."""
    m = FusedLinear(72, 136, activation="gelu", device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(rows, 72, generator=g, device="cuda").to(given).requires_grad_(True)
    r = torch.randn(rows, 136, generator=g, device="cuda", requires_grad=True)
    low = [t.detach().to(dt).requires_grad_(True) for t in (x, m.weight, m.bias)]
    for residual, out_dtype in ((None, dt), (r, torch.float32), (r.detach().to(dt), dt)):
        with torch.autocast("cuda", dt):
            out = m(x, residual)
        want = linear_act(*low, residual, activation="gelu", output_dtype=out_dtype)
        assert out.dtype == out_dtype and torch.equal(out, want)
        up = torch.randn(out.shape, generator=g, device="cuda").to(out_dtype)
        grads = torch.autograd.grad(out, (x, m.weight, m.bias), up)
        for got, ref, t in zip(grads, torch.autograd.grad(want, low, up), (x, m.weight, m.bias)):
            assert got.dtype == t.dtype and torch.equal(got, ref.to(t.dtype))
