"""The operators around the layer, without a GPU: plain forms, fallbacks, refusals at the C ABI, the optimizer's state."""

import ctypes
import io

import pytest
import torch

from mhc_mlx_amd import AdamW, FusedLinear, _lib, adamw_step_hip, linear_act, policy_loss
from mhc_mlx_amd import layer as L
from mhc_mlx_amd.linear import ACTIVATIONS, linear_act_reference
from mhc_mlx_amd.optim import BLOCK, _decode, _encode, adamw_step_reference
from tests._train import act64, policy64


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libmhc_hip.so not built")
    return _lib.load()


@pytest.mark.parametrize("act", ACTIVATIONS)
def test_plain_linear_act_and_its_gradient(act):
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 7), (6, 7), (6,), (5, 6)))
    y, d = act64(x @ w.t() + b, act)
    assert torch.allclose(linear_act_reference(x, w, b, r, act), y + r, rtol=1e-12, atol=1e-12)
    xx = x.clone().requires_grad_(True)
    up = torch.randn(5, 6, generator=g, dtype=torch.float64)
    linear_act_reference(xx, w, b, r, act).backward(up)
    assert torch.allclose(xx.grad, (up * d) @ w, rtol=1e-10, atol=1e-10)


def test_policy_formula_against_autograd_and_differences():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(12, 9, generator=g, dtype=torch.float64, requires_grad=True)
    a = torch.randint(0, 9, (12,), generator=g)
    lp = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    old, ref = (lp.detach() + 0.4 * torch.randn(12, generator=g) for _ in range(2))
    adv, w = torch.randn(12, generator=g), torch.rand(12, generator=g)
    w[3] = 0
    ratio = torch.exp(lp - old)
    each = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.3) * adv) + 0.2 * (torch.exp(ref - lp) - (ref - lp) - 1)
    loss = (w * each).sum() / w.sum()
    loss.backward()
    got, logp, c = policy64(z, a, old, adv, ref, w, 0.2, 0.3, 0.2)
    assert abs(float(got) - float(loss.detach())) < 1e-6 and logp[3] == 0
    hot = torch.nn.functional.one_hot(a, 9)
    assert torch.allclose(c[:, None] * (hot - torch.softmax(z.detach(), 1)), z.grad, atol=1e-7)


def test_fused_linear_falls_back_on_the_cpu(monkeypatch):
    monkeypatch.setattr(L, "_METAL_FAILED", True)  # (the warning has been given)
    m = FusedLinear(8, 6, activation="gelu")
    x = torch.randn(3, 8)
    assert torch.allclose(m(x), torch.nn.functional.gelu(torch.nn.functional.linear(x, m.weight, m.bias)), atol=1e-6)
    assert m(x, torch.ones(3, 6)).shape == (3, 6) and "gelu" in repr(m)
    assert set(m.state_dict()) == {"weight", "bias"}
    with pytest.raises(ValueError):
        FusedLinear(8, 6, activation="swish")


def test_fused_linear_under_autocast_on_the_cpu(monkeypatch):
    """As nn.Linear: operands in the autocast dtype, whatever x's; a float32 residual keeps its precision."""
    monkeypatch.setattr(L, "_METAL_FAILED", True)
    m = FusedLinear(32, 24)
    plain = torch.nn.Linear(32, 24)
    plain.load_state_dict(m.state_dict())
    r = torch.randn(5, 24)
    for x in (torch.randn(5, 32), torch.randn(5, 32).to(torch.bfloat16)):
        with torch.autocast("cpu", torch.bfloat16):
            y, z, with_r = m(x), plain(x), m(x, r)
        assert y.dtype == z.dtype == torch.bfloat16 and with_r.dtype == torch.float32
        low = [t.detach().to(torch.bfloat16).double() for t in (x, m.weight, m.bias)]
        exact = low[0] @ low[1].t() + low[2]
        assert bool(((y.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 1e-5).all())  # one rounding to bf16
        assert bool(((with_r.double() - exact - r).abs() <= 1e-5).all())  # fp32 sums of 32 products of size 1
        y.float().sum().backward()
        assert m.weight.grad.dtype == torch.float32
    with torch.autocast("cpu", torch.bfloat16):
        assert linear_act_reference(x.float(), m.weight).dtype == torch.float32


def test_operators_never_fall_back():
    x = torch.randn(3, 8)
    if not _lib.LIB_PATH.exists():
        pytest.skip("libmhc_hip.so not built")
    with pytest.raises(ValueError, match="GPU"):
        linear_act(x, torch.randn(4, 8))
    with pytest.raises(ValueError, match="GPU"):
        policy_loss(x, torch.zeros(3, dtype=torch.long), torch.zeros(3), torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        adamw_step_hip([x], [x], [x], [x], step=1)


def test_codes_round_trip():
    g = torch.Generator().manual_seed(2)
    t = torch.randn(1000, generator=g) * torch.exp(3 * torch.randn(1000, generator=g))
    codes, unit = _encode(t)
    assert codes.dtype == torch.float8_e4m3fn and unit.shape == (4,)
    back, u = _decode(codes, unit), unit.repeat_interleave(BLOCK)[:1000]
    assert bool(((back - t).abs() <= (2.0 ** -4 + 1e-6) * t.abs() + 2.0 ** -10 * u).all())
    again, same = _encode(back)
    assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8)) and torch.allclose(same, unit, rtol=1e-6)
    codes, unit = _encode(torch.zeros(300))
    assert not codes.float().any() and bool((unit > 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_follows_torchs(bits):
    """Against torch.optim.AdamW: in 32 bits up to rounding, in 8 as near as the states' codes let it."""
    torch.manual_seed(0)
    w = torch.randn(40, 120)
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    mine = AdamW([a], lr=1e-2, weight_decay=0.1, state_bits=bits)
    theirs = torch.optim.AdamW([b], lr=1e-2, weight_decay=0.1)
    for _ in range(20):
        g = torch.randn(40, 120)
        a.grad, b.grad = g.clone(), g.clone()
        mine.step()
        theirs.step()
    moved = (b.detach() - w).norm()
    assert (a.detach() - b.detach()).norm() < (1e-5 if bits == 32 else 0.1) * moved


def test_optimizer_state_keeps_its_types_through_a_checkpoint():
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(100, 64).to(torch.bfloat16)), torch.nn.Parameter(torch.randn(4))]
    opt = AdamW(ps, state_bits=8)
    for p in ps:
        p.grad = torch.randn_like(p)
    opt.step()
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf)
    buf.seek(0)
    fresh = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=8)
    fresh.load_state_dict(torch.load(buf, weights_only=True))
    for p, q in zip(ps, fresh.param_groups[0]["params"]):
        s, t = opt.state[p], fresh.state[q]
        assert set(s) == set(t) and s["step"] == t["step"] == 1
        for k in s:
            if k != "step":
                assert s[k].dtype == t[k].dtype and torch.equal(s[k].float(), t[k].float()) and s[k].data_ptr() != t[k].data_ptr()
    assert opt.state[ps[0]]["exp_avg"].dtype == torch.float8_e4m3fn and opt.state[ps[0]]["master"].dtype == torch.float32
    assert opt.state[ps[1]]["exp_avg"].dtype == torch.float32 and "master" not in opt.state[ps[1]]


def test_optimizer_and_step_refusals():
    p = torch.nn.Parameter(torch.randn(4))
    for bad in (dict(lr=-1), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(ValueError):
        adamw_step_reference([p], [p], [p], [p], step=0)


def test_adamw_rejects_bad_arguments_on_the_host(lib):
    def step(t, dtype=0, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, n=1, count=1):
        arr = (_lib.AdamWTensor * 1)(t) if t is not None else None
        return lib.mhc_adamw_step(arr, count, dtype, bits, lr, b1, b2, eps, wd, n, 1.0, None, None)

    T = lambda **k: _lib.AdamWTensor(**(dict(param=16, grad=16, exp_avg=16, exp_avg_sq=16, numel=4) | k))  # noqa: E731
    assert step(None, count=0) == 0
    assert step(T(numel=0)) == 0
    for bad in [dict(t=None), dict(t=T(param=None)), dict(t=T(grad=None)), dict(t=T(exp_avg=None)), dict(t=T(), bits=8), dict(t=T(), bits=4),
                dict(t=T(), dtype=3), dict(t=T(master=16)), dict(t=T(numel=-1)), dict(t=T(numel=1 << 60)), dict(t=T(), n=0), dict(t=T(), b1=1.0),
                dict(t=T(), lr=float("nan")), dict(t=T(), count=-1)]:
        assert step(**bad) == -1, bad
        assert lib.mhc_last_error()


def test_policy_rejects_bad_arguments_on_the_host(lib):
    def args(**k):
        base = dict(logits=16, row_stride=8, actions=16, old_logp=16, advantages=16, T=2, V=8, dtype=1)
        return _lib.PolicyArgs(**(base | k))

    def fwd(a, ws=16, nb=1 << 20):
        return lib.mhc_policy_loss_fwd(ctypes.byref(a) if a else None, 16, 16, 16, ws, nb, None)

    for bad in [None, args(logits=None), args(actions=None), args(T=-1), args(V=0), args(V=1 << 31), args(dtype=3), args(row_stride=7),
                args(clip_low=-1.0), args(denominator=-1.0), args(weights=16, weights_dtype=2)]:
        assert fwd(bad) == -1
        assert lib.mhc_last_error()
    assert fwd(args(), None) == -1 and fwd(args(), 16, 7) == -1
    assert lib.mhc_policy_loss_bwd(ctypes.byref(args()), None, None, 16, None) == -1
    assert lib.mhc_policy_loss_bwd(ctypes.byref(args(T=0)), None, None, None, None) == 0
    assert lib.mhc_policy_loss_fwd_bwd(ctypes.byref(args()), 1.0, 16, 16, None, 16, 1 << 20, None) == -1
    assert lib.mhc_policy_loss_workspace_bytes(-1) == 0


def test_linear_rejects_bad_arguments_on_the_host(lib):
    def fwd(x=16, ldx=64, w=16, ldw=64, out=16, odt=1, act=0, M=2, N=8, K=64, dt=1):
        return lib.mhc_linear_act_fwd(x, ldx, w, ldw, None, None, out, odt, None, act, M, N, K, dt, None, 0, None)

    assert fwd(M=0) == 0
    for bad in [dict(x=None), dict(w=None), dict(out=None), dict(M=-1), dict(N=0), dict(K=0), dict(dt=3), dict(odt=2), dict(act=5), dict(act=-1),
                dict(ldx=63), dict(ldw=63), dict(K=1 << 23)]:
        assert fwd(**bad) == -1, bad
        assert lib.mhc_last_error()

    def bwd(g=16, gdt=1, x=16, w=16, dx=16, dw=16, db=16, ldx=64, M=2, ws=256, nb=1 << 30):
        return lib.mhc_linear_act_bwd(g, gdt, None, x, ldx, w, 64, dx, dw, db, M, 8, 64, 1, ws, nb, None)

    for bad in [dict(g=None), dict(x=None), dict(w=None), dict(gdt=2), dict(ldx=63), dict(M=0), dict(ws=None), dict(nb=0), dict(ws=257)]:
        assert bwd(**bad) == -1, bad
    assert lib.mhc_linear_act_bwd_workspace_bytes(16, 1, None, 16, 64, 16, 64, 1, 1, 1, 0, 8, 64, 1) == 0
