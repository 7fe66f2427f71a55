"""The norm, the int8 rows and the cross entropy without a GPU: plain forms, formulas against differences, fallbacks, refusals at the C ABI."""

import ctypes

import pytest
import torch
import torch.nn as nn

from mhc_mlx_amd import AddRMSNorm, AutoPatcher, FusedLinear, Int8Linear, Int8Rows, MHCRewire, _lib, add_rms_norm, linear_cross_entropy, linear_int8, quantize_int8
from mhc_mlx_amd import layer as L
from mhc_mlx_amd.cross_entropy import linear_cross_entropy_reference
from mhc_mlx_amd.int8 import linear_int8_reference, quantize_int8_reference
from mhc_mlx_amd.norm import add_rms_norm_reference
from tests._block import ce64, check_codes, int8_product64, norm64, norm_grads64
from tests._train import close


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libmhc_hip.so not built")
    return _lib.load()


def rand(seed, *shapes, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g, dtype=dtype) for s in shapes]


def differences(f, t, up):
    """d <f, up> / dt by central differences."""
    out, flat, step = torch.zeros_like(t).view(-1), t.view(-1), 1e-6
    for k in range(flat.numel()):
        held = float(flat[k])
        flat[k] = held + step
        a = float((f() * up).sum())
        flat[k] = held - step
        b = float((f() * up).sum())
        flat[k] = held
        out[k] = (a - b) / (2 * step)
    return out.view(t.shape)


def test_norm_formula_against_autograd_and_differences():
    x, w, dy, dh = rand(0, (5, 9), (9,), (5, 9), (5, 9))
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, h = add_rms_norm_reference(xs, xs * 0, ws, 1e-3)
    torch.autograd.backward([y, h], [dy, dh])
    z, s = x, 1 / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-3)
    (dx, _), (dw, _) = norm_grads64(None, z, s, 0.0, w, dy, dh, torch.float32, torch.float32)
    assert torch.allclose(xs.grad, dx, rtol=1e-10, atol=1e-12) and torch.allclose(ws.grad, dw, rtol=1e-10, atol=1e-12)
    plain = lambda: add_rms_norm_reference(x, None, w, 1e-3)[0]  # noqa: E731
    assert torch.allclose(differences(plain, x, dy) + dh, dx, atol=1e-7)
    assert torch.allclose(differences(plain, w, dy), dw, atol=1e-7)


def test_cross_entropy_formula_against_autograd_and_differences():
    x, w = rand(1, (7, 5), (6, 5))
    y, m = torch.tensor([0, 5, 2, -100, 3, 1, 4]), torch.tensor([1.0, 0.5, 0.0, 1.0, -0.25, 2.0, 1.0])
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, logp = linear_cross_entropy_reference(xs, ws, y, m)
    loss.backward()
    r = ce64(x.float(), w.float(), y, m)
    live = torch.where(y == -100, 0.0, m) != 0
    lp = torch.log_softmax(x @ w.t(), 1)[torch.arange(7), y.clamp(min=0)]
    assert torch.allclose(logp, torch.where(live, lp, 0.0)) and torch.allclose(loss.detach(), -(m * lp)[live].sum() / m[live].sum())
    assert abs(float(loss.detach()) - float(r["loss"][0])) < 1e-6 and float((xs.grad - r["dx"][0]).abs().max()) < 1e-6
    assert float((ws.grad - r["dw"][0]).abs().max()) < 1e-6
    plain = lambda: linear_cross_entropy_reference(x, w, y, m)[0]  # noqa: E731
    one = torch.ones((), dtype=torch.float64)
    assert torch.allclose(differences(plain, x, one), xs.grad, atol=1e-7) and torch.allclose(differences(plain, w, one), ws.grad, atol=1e-7)
    none = linear_cross_entropy_reference(x, w, y, torch.zeros(7))
    assert float(none[0]) == 0 and not none[1].any()
    assert bool(linear_cross_entropy_reference(x, w, torch.full((7,), 6))[0].isnan())


def test_plain_int8_rows_and_product():
    x, w, b, r = rand(2, (4, 3, 33), (10, 33), (10,), (4, 3, 10), dtype=torch.float32)
    q, p = quantize_int8_reference(x), quantize_int8_reference(w)
    check_codes(q.codes, q.scales, x.double(), 0.0)
    assert float((q.dequantize() - x).abs().max()) <= 0.5001 * float(q.scales.max()) and q.dequantize(torch.bfloat16).dtype == torch.bfloat16
    for act in ("none", "gelu", "silu"):
        close(linear_int8_reference(q, p, b, r, act, torch.float32), *int8_product64(q, p, b, r, act, torch.float32))
    odd = torch.tensor([[0.0, 0.0], [1.0, float("inf")], [float("nan"), 1.0]])
    z = quantize_int8_reference(odd)
    assert z.scales[0] == 0 and bool(z.scales[1:].isnan().all()) and not z.codes.any()


def test_modules_fall_back_on_the_cpu(monkeypatch):
    monkeypatch.setattr(L, "_METAL_FAILED", True)  # (the warning has been given)
    x, r = rand(3, (6, 16), (6, 16), dtype=torch.float32)
    norm = AddRMSNorm(16)
    y, h = norm(x, r)
    want = (x + r) * torch.rsqrt((x + r).square().mean(1, keepdim=True) + norm.eps)
    assert torch.equal(h, x + r) and torch.allclose(y, want, atol=1e-6) and set(norm.state_dict()) == {"weight"}
    lin = FusedLinear(16, 16, activation="gelu")
    q = Int8Linear.from_linear(lin)
    rows, _ = AddRMSNorm(16, int8=True)(x)
    assert isinstance(rows, Int8Rows) and q(rows).dtype == torch.float32
    assert float((q(x) - lin(x)).detach().abs().max()) < 0.05 and "gelu" in repr(q) and "int8" in repr(AddRMSNorm(4, int8=True))
    assert set(q.state_dict()) == {"weight", "weight_scale", "bias"} and Int8Linear(4, 4, bias=False).bias is None
    half = Int8Linear.from_linear(FusedLinear(16, 16).to(torch.bfloat16)).half()
    assert half.weight_scale.dtype == half.bias.dtype == torch.float32 and half.return_dtype == torch.bfloat16
    model = nn.ModuleList([half, Int8Linear(16, 8)])
    assert AutoPatcher.patch(model, n_streams=4, verbose=False) == 1 and isinstance(model[0], MHCRewire)
    with torch.no_grad():
        assert model[0](x.to(torch.bfloat16)).dtype == torch.bfloat16


def test_argument_checks_without_a_gpu():
    x = torch.zeros(2, 4)
    for eps in (0.0, -1.0, float("inf"), float("nan"), 1e-45):
        with pytest.raises(ValueError, match="eps"):
            add_rms_norm(x, eps=eps)
    with pytest.raises(ValueError, match="denominator"):
        linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.long), denominator=0.0)
    with pytest.raises(ValueError, match="activation"):
        linear_int8(quantize_int8_reference(x), quantize_int8_reference(x), activation="tanh")
    for call in (lambda: add_rms_norm(x), lambda: quantize_int8(x), lambda: linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.long)),
                 lambda: linear_int8(quantize_int8_reference(x), quantize_int8_reference(x))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_norm_refusals_at_the_c_abi(lib):
    p, eps = ctypes.c_void_p(4096), ctypes.c_float(1e-6)  # never dereferenced: every call below is rejected on the host

    def fwd(x=p, ldx=8, r=None, ldr=8, w=p, wd=0, h=None, y=p, T=2, C=8, dt=0, e=eps):
        return lib.mhc_add_rms_norm_fwd(x, ldx, r, ldr, w, wd, h, y, None, T, C, dt, e, None)

    def int8(x=p, ldx=8, r=None, ldr=8, w=p, wd=0, h=None, y=p, s=p, T=2, C=8, dt=0, e=eps):
        return lib.mhc_add_rms_norm_int8(x, ldx, r, ldr, w, wd, h, y, s, T, C, dt, e, None)

    for f in (fwd, int8):
        for bad in (dict(T=-1), dict(C=0), dict(C=1 << 24), dict(dt=3), dict(wd=1), dict(x=None), dict(y=None), dict(r=p), dict(ldx=7),
                    dict(r=p, h=p, ldr=7), dict(e=ctypes.c_float(0.0)), dict(e=ctypes.c_float(float("nan")))):
            assert f(**bad) == -1, bad
        assert f(T=0, x=None, y=None) == 0
    assert int8(s=None) == -1 and b"null" in lib.mhc_last_error()
    assert lib.mhc_quantize_int8(None, 8, p, p, 2, 8, 0, None) == -1 and lib.mhc_quantize_int8(p, 7, p, p, 2, 8, 0, None) == -1
    assert lib.mhc_quantize_int8(None, 8, None, None, 0, 8, 0, None) == 0
    for bad in ((None, 8, p, p, 1, 2, 8), (p, 8, None, p, 1, 2, 8), (p, 8, p, None, 1, 2, 8), (p, 7, p, p, 1, 2, 8), (p, 8, p, p, 3, 2, 8), (p, 8, p, p, 1, 2, 0)):
        assert lib.mhc_dequantize_int8(*bad, None) == -1
    assert lib.mhc_dequantize_int8(None, 8, None, None, 1, 0, 8, None) == 0
    nb = lib.mhc_add_rms_norm_bwd_workspace_bytes(100, 64, 1)
    assert nb > 0 and lib.mhc_add_rms_norm_bwd_workspace_bytes(0, 64, 1) == 0

    def bwd(dy=p, lddy=64, h=p, rstd=p, w=p, wd=1, dw=p, ws=p, n=nb, T=100, dt=1):
        return lib.mhc_add_rms_norm_bwd(dy, lddy, None, 0, h, 64, rstd, w, wd, None, dw, T, 64, dt, ws, n, None)

    for bad in (dict(T=0), dict(dy=None), dict(h=None), dict(rstd=None), dict(lddy=63), dict(wd=2), dict(ws=None), dict(n=nb - 1), dict(dt=7),
                dict(ws=ctypes.c_void_p(4100))):
        assert bwd(**bad) == -1, bad
    assert bwd(dw=None, w=None) == 0  # nothing asked for


def test_int8_refusals_at_the_c_abi(lib):
    p = ctypes.c_void_p(4096)

    def call(x=p, ldx=32, xs=p, w=p, ldw=32, ws=p, out=p, od=1, act=0, M=100, N=8, K=32, buf=None, n=0):
        return lib.mhc_linear_int8(x, ldx, xs, w, ldw, ws, None, None, out, od, act, M, N, K, buf, n, None)

    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(M=1 << 28), dict(N=1 << 22), dict(M=1 << 27, N=1 << 21), dict(K=1 << 17, ldx=1 << 17, ldw=1 << 17), dict(od=3), dict(act=5),
                dict(act=-1), dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(ldx=31), dict(ldw=31)):
        assert call(**bad) == -1, bad
    assert call(M=0, x=None) == 0
    odd = lib.mhc_linear_int8_workspace_bytes(p, 33, p, 33, 100, 8, 33)
    assert odd >= 108 * 48 and call(ldx=33, ldw=33, K=33, buf=p, n=odd - 1) == -1 and call(ldx=33, ldw=33, K=33, buf=ctypes.c_void_p(4100), n=odd) == -1
    assert lib.mhc_linear_int8_workspace_bytes(p, 1 << 17, p, 1 << 17, 100, 8, 1 << 17) == 0


def test_cross_entropy_refusals_at_the_c_abi(lib):
    p = ctypes.c_void_p(4096)

    def args(**kw):
        a = dict(x=p, ldx=16, w=p, ldw=16, targets=p, weights=None, weights_dtype=0, T=10, V=20, C=16, dtype=1, ignore_index=-100, denominator=0.0)
        return _lib.LinearCeArgs(**{**a, **kw})

    def fwd(a, loss=p, logp=p, state=p, ws=p, n=1 << 40):
        return lib.mhc_linear_ce_fwd(ctypes.byref(a) if a else None, loss, logp, state, ws, n, None)

    def bwd(a, state=p, dx=p, dw=p, ws=p, n=1 << 40):
        return lib.mhc_linear_ce_bwd(ctypes.byref(a) if a else None, state, None, ctypes.c_float(1.0), dx, dw, ws, n, None)

    for kw in (dict(T=-1), dict(V=0), dict(C=0), dict(T=1 << 28), dict(V=1 << 22), dict(C=1 << 22), dict(T=1 << 27, V=1 << 21), dict(dtype=3), dict(denominator=-1.0), dict(x=None),
               dict(w=None), dict(targets=None), dict(ldx=15), dict(ldw=15), dict(weights=p, weights_dtype=1)):
        assert fwd(args(**kw)) == -1 and bwd(args(**kw)) == -1, kw
    a = args()
    kept = lambda **kw: lib.mhc_linear_ce_logits_bytes(ctypes.byref(args(**kw)))  # noqa: E731
    assert kept(C=1024) == kept(C=256, dtype=0) == 10 * 64 * 4 and kept() == 0 and lib.mhc_linear_ce_logits_bytes(None) == 0
    assert kept(T=1 << 14, V=1 << 15, C=1024) == 1 << 31 and kept(T=1 << 14, V=(1 << 15) + 1, C=1024) == 0
    assert fwd(args(logits=4100)) == -1 and bwd(args(logits=4100)) == -1
    nf, nb = lib.mhc_linear_ce_fwd_workspace_bytes(ctypes.byref(a)), lib.mhc_linear_ce_bwd_workspace_bytes(ctypes.byref(a), 1, 1)
    assert nf > 0 and nb > 0 and lib.mhc_linear_ce_state_bytes(10) >= 24 * 10
    off = ctypes.c_void_p(4100)
    for kw in (dict(loss=None), dict(logp=None), dict(state=None), dict(ws=None), dict(n=nf - 1), dict(state=off), dict(ws=off)):
        assert fwd(a, **kw) == -1, kw
    for kw in (dict(state=None), dict(ws=None), dict(n=nb - 1), dict(state=off), dict(ws=off)):
        assert bwd(a, **kw) == -1, kw
    assert fwd(None) == -1 and bwd(None) == -1 and bwd(args(T=0)) == -1
    assert bwd(a, dx=None, dw=None) == 0
    assert lib.mhc_linear_ce_fwd_workspace_bytes(None) == 0 and lib.mhc_linear_ce_bwd_workspace_bytes(None, 1, 1) == 0
