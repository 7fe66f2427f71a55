"""linear_act / FusedLinear at the ends of what they take: very long rows, many rows, tiny values, mixed types."""

import pytest
import torch

from tests._train import U32, UNIT, act64, close, linear64, linear_grads64

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


def _holed(t, fill, pad=12):
    """t's values in rows `pad` elements longer, whose extra elements are `fill`."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), fill, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


# fp32 sizes whose products, of the call and of its backward, are summed in tiles of every height and width from 64 x 128 on
SPLIT = [(2048, 2048, 104), (1000, 1100, 1540), (2048, 2048, 2048), (1500, 2048, 4100), (4096, 4096, 264), (6000, 6000, 1100)]


def _normal(seed, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda") * (s[-1] ** -0.5 if len(s) == 2 and k == 1 else 1.0) for k, s in enumerate(shapes)]


@pytest.mark.parametrize("M,N,K", SPLIT)
def test_fp32_results_do_not_depend_on_what_lies_between_rows(M, N, K):
    x, w, g = _normal(8, (M, K), (N, K), (M, N))
    runs = []
    for fill in (0.0, float("nan"), float("inf")):
        ts = [_holed(t, fill).requires_grad_(True) for t in (x, w)]
        out = linear_act(*ts)
        runs.append((out.detach(), *torch.autograd.grad(out, ts, g)))
    assert all(torch.equal(p, q) for run in runs[1:] for p, q in zip(run, runs[0]))


@pytest.mark.parametrize("M,N,K", SPLIT)
def test_fp32_results_do_not_depend_on_other_rows(M, N, K):
    """Bit by bit: NaN and infinities in some rows of every operand leave every other sum as it was."""
    x, w, g = _normal(9, (M, K), (N, K), (M, N))
    rows, cols = torch.tensor([1, M // 2, M - 1], device="cuda"), torch.tensor([0, N - 3], device="cuda")
    x2, w2 = x.clone(), w.clone()
    x2[1, K // 2], x2[M // 2, 0], x2[M - 1, K - 1] = float("nan"), float("inf"), -float("inf")
    w2[0, K - 1], w2[N - 3, 1] = float("inf"), float("nan")
    clean, out = linear_act(x, w), linear_act(x2, w2)
    keep = torch.ones_like(clean, dtype=torch.bool)
    keep[rows], keep[:, cols] = False, False
    assert torch.equal(out[keep], clean[keep])
    ref = x2.double() @ w2.double().t()
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(out.isinf(), ref.isinf())
    assert torch.equal(out[out.isinf()].sign().double(), ref[ref.isinf()].sign())
    # dx = g W: a row of g; dW = g^T x: a column of g and a column of x
    ts = [t.requires_grad_(True) for t in (x, w)]
    y = linear_act(*ts)
    dx, dw = torch.autograd.grad(y, ts, g, retain_graph=True)
    g2 = g.clone()
    g2[3, 5] = float("nan")
    dx2, dw2 = torch.autograd.grad(y, ts, g2)
    assert dx2[3].isnan().all() and dw2[5].isnan().all()
    dx2[3], dw2[5] = dx[3], dw[5]
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("M,N,K", [(5, 64, 96), (100, 130, 96)] + SPLIT)
def test_fp32_values_near_both_ends_of_the_range(M, N, K):
    """Rows of values down to subnormal ones against weights that make ordinary numbers of them, and large results."""
    x, w = _normal(10, (M, K), (N, K))
    for row, size in ((0, 1e-34), (1, 1e-36), (2, 1e-37), (3, 1e-39), (M - 1, 1e30)):
        x[row] *= size
    w[1::2] *= 1e36
    w[2] *= 1e-36
    out = linear_act(x, w)
    ref, bound, *_ = linear64(x, w, None, None, "none", torch.float32)
    fine = ref.abs() < 3e38
    close(torch.where(fine, out.double(), 0.0), torch.where(fine, ref, 0.0), torch.where(fine, bound, 1.0), "out")
    assert not out[:4].isinf().any()


def test_fp32_gradients_of_tiny_values():
    """Both products of the backward with a gradient that is as small, in tiles of several sizes."""
    for M, N, K in SPLIT:
        x, w, g = _normal(11, (M, K), (N, K), (M, N))
        x, w, g = x * 1e30, w * 1e28, g * 1e-37
        ts = [t.requires_grad_(True) for t in (x, w)]
        dx, dw = torch.autograd.grad(linear_act(*ts), ts, g)
        one = torch.ones(M, N, dtype=torch.float64, device="cuda")
        px, pw, _ = linear_grads64(x, w, g, one, torch.zeros_like(one), torch.float32, False)
        close(dx, *px, f"dx {M} {N} {K}")
        close(dw, *pw, f"dw {M} {N} {K}")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [3, 300])
def test_gradients_of_units_far_below_zero(act, dt, M):
    """act' keeps its precision where it is small: x is 0, so that z is the bias and db a sum of equal values."""
    b = torch.linspace(-14, 8, 1001, device="cuda").to(dt).requires_grad_(True)
    x, w = torch.zeros(M, 16, device="cuda", dtype=dt), torch.ones(1001, 16, device="cuda", dtype=dt)
    out = linear_act(x, w, b, activation=act)
    db, = torch.autograd.grad(out, b, torch.ones_like(out))
    z = b.detach().double()
    _, d = act64(z, act)
    # its code: 2^-10 of it, down to 2^-39; its formula: roundings of the exponent's argument (up to 2^7, 16 where act' is
    # above 2^-39) and a few more of each term, and the normal distribution's polynomial
    phi = torch.exp(-z * z / 2)
    terms = {"gelu": z.abs() * phi + torch.special.ndtr(z), "silu": torch.sigmoid(z) * (1 + z.abs()),
             "gelu_tanh": d.abs() + 4 * torch.sigmoid(1.6 * z + 0.0714 * z ** 3) * (1 + z.abs() ** 3)}[act]
    bound = 2.0 ** -10 * d.abs() + 2.0 ** -39 + 256 * U32 * terms + (7e-6 * torch.special.ndtr(z) if act == "gelu" else 0.0)
    close(db, M * d, M * bound + UNIT[dt] * M * d.abs() + 2.0 ** -25, act)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [3, 300])
def test_values_of_units_far_below_zero(act, dt, M):
    """float32 outputs hold 2^-14 of an activation however small it is."""
    b = torch.linspace(-9, 9, 1001, device="cuda").to(dt)
    x, w = torch.zeros(M, 16, device="cuda", dtype=dt), torch.ones(1001, 16, device="cuda", dtype=dt)
    z = b.double()
    y = z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5) if act == "gelu" else act64(z, act)[0]  # (ndtr is 1 + erf: 0 from -8.3 on)
    y = y.expand(M, 1001)
    # Phi's fit 7e-6; the exponent's argument, up to 75 (gelu_tanh at -9), rounded three times
    close(linear_act(x, w, b, activation=act, output_dtype=torch.float32), y, (7e-6 + 256 * U32 + 16 * U32) * y.abs() + 2.0 ** -126, act)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [3, 300])
def test_nan_goes_through_the_derivative(act, M):
    x, w, b, g = (t.to(torch.bfloat16) for t in _normal(12, (M, 40), (136, 40), (136,), (M, 136)))
    x[1, 7], b[5] = float("nan"), -float("nan")
    ts = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear_act(*ts, activation=act), ts, g)
    assert dx.isnan().all() and dw.isnan().all() and db.isnan().all()  # (every row has column 5, every column row 1)
    with torch.no_grad():
        b[5] = 0
    dx, _, db = torch.autograd.grad(linear_act(*ts, activation=act), ts, g)
    assert dx[1].isnan().all() and dx[[k for k in range(M) if k != 1]].isfinite().all() and db.isnan().all()
