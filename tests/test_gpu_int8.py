"""linear_int8 and Int8Linear on the GPU against float64 (tests/_block.py)."""

import pytest
import torch
import torch.nn as nn

from mhc_mlx_amd import (AddRMSNorm, AutoPatcher, FusedLinear, Int8Linear, Int8Rows, MHCRewire, add_rms_norm_int8, kernel_timer, linear_int8,
                         quantize_int8)
from mhc_mlx_amd import layer as L
from mhc_mlx_amd.int8 import linear_int8_reference, quantize_int8_reference
from mhc_mlx_amd.linear import ACTIVATIONS
from tests._block import int8_product64
from tests._train import close

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(g, *shape, low=-127):
    codes = torch.randint(low, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    return Int8Rows(codes, torch.rand(shape[:-1], generator=g, device="cuda") * 0.02 + 1e-3)


def check(g, M, N, K, dt, act="none", bias=True, residual=True):
    x, w = rows_of(g, M, K), rows_of(g, N, K)
    w = Int8Rows(w.codes, w.scales / K ** 0.5)
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    r = torch.randn(M, N, generator=g, device="cuda").to(dt) if residual else None
    out = linear_int8(x, w, b, r, act, dt)
    assert out.dtype == dt
    close(out, *int8_product64(x, w, b, r, act, dt), f"{M} {N} {K} {act}")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 16, 17, 33, 64, 65, 130, 300])
def test_products(dt, M):
    g = gen(M)
    for N, K in ((1, 1), (16, 64), (17, 3), (33, 128), (130, 132), (250, 1027), (64, 1024), (100, 260), (520, 2049)):
        check(g, M, N, K, dt, bias=N % 2 == 0, residual=K % 2 == 0)


@pytest.mark.parametrize("dt", DTYPES)
def test_values(dt):
    g = gen(2)
    for shape in ((1, 1), (3, 7), (2, 5, 64), (40, 1001), (9, 16384)):
        rows = rows_of(g, *shape, low=-128)
        want = rows.codes.float() * rows.scales[..., None]
        assert torch.equal(rows.dequantize(dt), want.to(dt)) and torch.equal(rows.dequantize(torch.float64), want.double())
    part = Int8Rows(rows.codes[:, 3:999], rows.scales)
    assert torch.equal(part.dequantize(dt), want[:, 3:999].to(dt))
    assert Int8Rows(rows.codes[:0], rows.scales[:0]).dequantize(dt).shape == (0, 16384)
    with pytest.raises(ValueError):
        rows.dequantize(torch.int32)
    with pytest.raises(ValueError):
        Int8Rows(rows.codes, rows.scales[:3]).dequantize(dt)


def test_results_carry_no_gradient():
    g = gen(3)
    x = torch.randn(4, 64, generator=g, device="cuda", requires_grad=True)
    w = rows_of(g, 8, 64)
    rows, h = add_rms_norm_int8(x.t().contiguous().t(), x, torch.ones(64, device="cuda", requires_grad=True))
    out = linear_int8(quantize_int8(x[:, ::2][:, :32].contiguous().repeat(1, 2)), w, torch.zeros(8, device="cuda", requires_grad=True),
                      torch.zeros(4, 8, device="cuda", requires_grad=True).t().contiguous().t(), output_dtype=torch.float32)
    assert not any(t.requires_grad for t in (rows.codes, rows.scales, h, out, rows.dequantize()))


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("dt", DTYPES)
def test_activations(act, dt):
    g = gen(1)
    for M in (3, 100):
        check(g, M, 90, 256, dt, act)
        check(g, M, 90, 256, dt, act, bias=False, residual=False)


@pytest.mark.parametrize("M,N,K", [(1024, 1030, 512), (257, 513, 4096), (70, 128, 16384), (2000, 256, 8192), (4096, 2048, 128), (128, 20000, 130)])
def test_every_tile_and_split(M, N, K):
    check(gen(M + N), M, N, K, torch.bfloat16, "gelu")
    check(gen(M + N + 1), M, N, K, torch.float32, residual=False)


@pytest.mark.parametrize("M", [1, 20, 64, 129, 700])
def test_sums_are_exact(M):
    """The largest codes over the longest rows: 2^31 - 2^14 without a rounding before the scales; and sums of both signs."""
    K = (1 << 17) - 1
    x = Int8Rows(torch.full((M, K), -128, dtype=torch.int8, device="cuda"), torch.ones(M, device="cuda"))
    w = Int8Rows(torch.full((20, K), -128, dtype=torch.int8, device="cuda"), torch.ones(20, device="cuda"))
    want = torch.tensor(float(K * 128 * 128)).float().item()
    out = linear_int8(x, w, output_dtype=torch.float32)
    assert bool(((out - want).abs() <= 2.0 ** 31 * 2.0 ** -24 * 17).all())  # (parts of the reduction are rounded one by one)
    g = gen(M)
    a, b = (torch.randint(-3, 4, (n, 1000), generator=g, device="cuda", dtype=torch.int8) for n in (M, 40))
    one = lambda n: torch.full((n,), 0.5, device="cuda")  # noqa: E731
    out = linear_int8(Int8Rows(a, one(M)), Int8Rows(b, one(40)), output_dtype=torch.float32)
    assert torch.equal(out.double(), (a.double() @ b.double().t()) / 4)


def test_strides_views_and_shapes():
    g = gen(4)
    wide = rows_of(g, 6, 5, 400).codes
    w = rows_of(g, 48, 128)
    for x in (wide[:, :, 4:132], wide[:, :, 3:131], wide[::2, 1, 8:136], wide.transpose(0, 1)[..., :128], wide[:, :, ::2][..., :128], wide[0, 0, :128]):
        s = torch.rand(2, *x.shape[:-1], generator=g, device="cuda")[0]
        a = linear_int8(Int8Rows(x, s), w)
        b = linear_int8(Int8Rows(x.contiguous(), s), w)
        assert a.shape == (*x.shape[:-1], 48) and torch.equal(a, b)
    ww = rows_of(g, 48, 300)
    x = rows_of(g, 100, 128)
    for codes in (ww.codes[:, 1:129], ww.codes[:, 4:132], ww.codes[:, :256:2]):
        assert torch.equal(linear_int8(x, Int8Rows(codes, ww.scales)), linear_int8(x, Int8Rows(codes.contiguous(), ww.scales)))
    r = torch.randn(48, 100, generator=g, device="cuda").to(torch.bfloat16).t()
    b = torch.randn(48, 2, generator=g, device="cuda").half()[:, 0]
    assert torch.equal(linear_int8(x, w, b, r), linear_int8(x, w, b.float().contiguous(), r.contiguous()))
    none = linear_int8(Int8Rows(torch.empty(0, 128, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda")), w)
    assert none.shape == (0, 48)


def test_scales_that_are_zero_or_nan_stay_in_their_row():
    g = gen(5)
    for M in (5, 200):
        x, w = rows_of(g, M, 96), rows_of(g, 70, 96)
        x.scales[1], x.scales[2] = 0.0, float("nan")
        out = linear_int8(x, w, output_dtype=torch.float32)
        assert not out[1].any() and bool(out[2].isnan().all())
        keep = torch.arange(M, device="cuda") != 2
        assert bool(out[keep].isfinite().all())


def test_refusals():
    g = gen(6)
    x, w = rows_of(g, 4, 32), rows_of(g, 8, 32)
    ok = torch.zeros(8, device="cuda")
    for a, b, kw in ((Int8Rows(x.codes.float(), x.scales), w, {}), (Int8Rows(x.codes, x.scales[:3]), w, {}), (Int8Rows(x.codes, x.scales.half()), w, {}),
                     (Int8Rows(x.codes[:, :31], x.scales), w, {}), (x, Int8Rows(w.codes, w.scales[None]), {}), (x, w, dict(bias=ok[:7])),
                     (x, w, dict(residual=torch.zeros(4, 8, device="cuda"))), (x, w, dict(activation="tanh")), (x, w, dict(output_dtype=torch.int8)),
                     (Int8Rows(x.codes.cpu(), x.scales.cpu()), w, {}), (x, w, dict(bias=torch.zeros(8)))):
        with pytest.raises(ValueError):
            linear_int8(a, b, **kw)
    long = Int8Rows(torch.zeros(2, 1 << 17, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="2\\^17"):
        linear_int8(long, long)


@pytest.mark.parametrize("dt", DTYPES)
def test_module_norm_and_rewire(dt, monkeypatch):
    """The operators as a block has them: norm, product, residual; and inside MHCRewire by AutoPatcher."""
    g = gen(7)
    lin = FusedLinear(256, 256, activation="silu", device="cuda", dtype=dt)
    q = Int8Linear.from_linear(lin)
    w = quantize_int8(lin.weight)
    assert torch.equal(q.weight, w.codes) and torch.equal(q.weight_scale, w.scales) and q.activation == "silu"
    norm = AddRMSNorm(256, int8=True, device="cuda", dtype=dt)
    x, r = (torch.randn(3, 20, 256, generator=g, device="cuda").to(dt) for _ in range(2))
    rows, h = norm(x, r)
    y = q(rows, h)
    want, _ = add_rms_norm_int8(x, r, norm.weight)
    assert y.dtype == dt and torch.equal(y, linear_int8(want, w, lin.bias, x + r, "silu", dt))
    assert torch.equal(q(x), linear_int8(quantize_int8(x), w, lin.bias, None, "silu", dt))
    low, full = q(x).double(), lin(x).detach().double()
    assert float((low - full).norm() / full.norm()) < 0.03  # (steps of 1/127 of a row's largest value, in both operands)
    with kernel_timer() as kt:
        assert torch.equal(q(x), low.to(dt))
    assert {"quantize_int8", "linear_int8"} <= set(kt.stats())
    q.to(torch.float16)
    assert q.weight_scale.dtype == q.bias.dtype == torch.float32 and torch.equal(q.weight_scale, w.scales)
    model = nn.Sequential(Int8Linear.from_linear(lin), nn.Linear(256, 8, device="cuda", dtype=dt))
    assert AutoPatcher.patch(model, n_streams=4, verbose=False) == 1 and isinstance(model[0], MHCRewire)
    with torch.no_grad():
        out = model(x.reshape(60, 256))
    assert out.shape == (60, 8) and bool(out.isfinite().all()) and not L._METAL_FAILED
    state = q.state_dict()
    other = Int8Linear(256, 256, activation="silu", device="cuda", return_dtype=dt)
    other.load_state_dict(state)
    assert torch.equal(other(x), q(x))


def test_module_falls_back_for_wide_layers(monkeypatch):
    monkeypatch.setattr(L, "_METAL_FAILED", True)  # (the warning has been given)
    K = 1 << 17
    m = Int8Linear(K, 3, device="cuda", return_dtype=torch.float32)
    m.weight.copy_(torch.randint(-127, 128, (3, K), device="cuda"))
    m.weight_scale.fill_(0.01)
    x = torch.randn(2, K, device="cuda")
    q = quantize_int8_reference(x)
    assert torch.equal(m(x), linear_int8_reference(q, Int8Rows(m.weight, m.weight_scale), m.bias, output_dtype=torch.float32))


def test_captured_calls():
    g = gen(8)
    x = torch.randn(33, 512, generator=g, device="cuda").to(torch.bfloat16)
    many = torch.randn(600, 512, generator=g, device="cuda").to(torch.bfloat16)
    m = Int8Linear.from_linear(FusedLinear(512, 1024, activation="gelu", device="cuda", dtype=torch.bfloat16))
    step = lambda: [m(x), m(many)]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
        step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(other, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        x.normal_(generator=g)
        many.normal_(generator=g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
