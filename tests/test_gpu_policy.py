"""GPU parity of policy_loss / policy_loss_and_grad with the formulas in float64 (tests/_train.py)."""

import math

import pytest
import torch

from tests._train import LEAST, U32, UNIT, close, policy64

from mhc_mlx_amd import kernel_timer, policy_loss, policy_loss_and_grad

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(T, V, dt, seed=0, masked=0.25):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * T + V)
    z = (2 * torch.randn(T, V, generator=g, device="cuda")).to(DT[dt])
    a = torch.randint(0, V, (T,), generator=g, device="cuda")
    lp = torch.log_softmax(z.double(), 1).gather(1, a[:, None])[:, 0].float()
    old, ref = (lp + s * torch.randn(T, generator=g, device="cuda") for s in (0.3, 0.4))
    adv = torch.randn(T, generator=g, device="cuda")
    mask = torch.rand(T, generator=g, device="cuda") >= masked
    return z, a, old, adv, ref, mask


def _check(z, a, old, adv, ref=None, mask=None, lo=0.2, hi=0.3, kl=0.0, den=None, scale=1.0):
    """Loss, logp and gradient of both forms."""
    T, V = z.shape
    loss64, lp64, c64 = policy64(z, a, old, adv, ref, mask, lo, hi, kl, den)
    w = torch.ones(T, device="cuda", dtype=torch.float64) if mask is None else mask.double()
    on = w != 0
    D = den or float(w.cpu().sum()) or 1.0
    top = z.double().abs().nan_to_num(0, 0, 0).amax(1) if T else z.new_zeros(0).double()
    # the sum of exponentials: its terms' arguments and the additions of a thread and over threads; then z - top - log
    lp_off = (V / 512 + 64) * U32 + 4 * U32 * (top + 32)
    r = torch.exp(lp64 - old.double())
    size = r * adv.double().abs()  # how far coef and the loss move for a step of lp, and their roundings
    if ref is not None:
        size = size + kl * (1 + torch.exp(ref.double() - lp64))
    off = torch.where(on, w.abs() * size * (1.1 * lp_off + 16 * U32 * (1 + old.double().abs())), torch.zeros_like(size)) / D
    kw = dict(ref_logp=ref, mask=mask, clip_low=lo, clip_high=hi, kl_coef=kl, denominator=den)
    zz = z.detach().requires_grad_(True)
    loss, logp = policy_loss(zz, a, old, adv, **kw)
    assert loss.shape == () and loss.dtype == logp.dtype == torch.float32 and not logp.requires_grad
    loss_bound = off.cpu().sum() + (T / 512 + 64) * U32 * (torch.where(on, w.abs() * size, torch.zeros_like(size)).cpu().sum() / D + abs(float(loss64)))
    close(logp, lp64, torch.where(on, lp_off, torch.zeros_like(lp_off)) + U32 * lp64.abs(), "logp")
    close(loss.cpu(), loss64.cpu(), loss_bound, "loss")
    g, = torch.autograd.grad(loss, zz, torch.tensor(scale, device="cuda"))
    loss2, logp2, g2 = policy_loss_and_grad(z, a, old, adv, **kw, grad_scale=scale)
    close(loss2.cpu(), loss64.cpu(), loss_bound, "loss")
    close(logp2, lp64, torch.where(on, lp_off, torch.zeros_like(lp_off)) + U32 * lp64.abs(), "logp")
    p = torch.softmax(torch.where(on[:, None], z.double(), 0.0), 1)
    hot = torch.zeros_like(p)
    hot[torch.arange(T, device="cuda"), torch.where(on, a, 0).long()] = 1
    ref_g = scale * c64[:, None] * (hot - p)
    bound = scale * (off[:, None] + c64.abs()[:, None] * (lp_off[:, None] + 8 * U32)) * (hot + p) + UNIT[z.dtype] * 1.01 * ref_g.abs() + LEAST[z.dtype]
    # an exponential below the least normal number is taken as 0
    bound = bound + scale * c64.abs()[:, None] * 2.0 ** -125
    for got, what in ((g, "autograd"), (g2, "fused")):
        assert got.dtype == z.dtype
        close(got, ref_g, bound, what)
        assert not got[~on].any()


@pytest.mark.parametrize("T,V", [(1, 1), (1, 2), (3, 7), (5, 8), (2, 1000), (17, 1023), (33, 1025), (64, 4096), (9, 8191), (4, 16384),
                                 (7, 32003), (3, 65536), (2, 65537), (2, 131072), (2, 131080), (1, 200001), (700, 257)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_sizes(T, V, dt):
    z, a, old, adv, ref, mask = _inputs(T, V, dt)
    _check(z, a, old, adv, ref, mask, kl=0.1, scale=1024.0 if dt == "f16" else 1.0)


@pytest.mark.parametrize("kl,with_ref", [(0.0, False), (0.0, True), (0.5, True)])
@pytest.mark.parametrize("mask", ["none", "bool", "weights"])
@pytest.mark.parametrize("den", [None, 37.5])
def test_options(kl, with_ref, mask, den):
    z, a, old, adv, ref, m = _inputs(50, 300, "bf16", 1)
    weights = {"none": None, "bool": m, "weights": m.float() * torch.rand(50, device="cuda")}[mask]
    _check(z, a, old, adv, ref if with_ref else None, weights, 0.1, 0.4, kl, den)


def test_more_rows_than_workgroups_at_once():
    z, a, old, adv, ref, mask = _inputs(20000, 33, "bf16", 2)
    _check(z, a, old, adv, ref, mask, kl=0.1)


@pytest.mark.parametrize("vecs", [1025, 4096, 4097, 6656, 6657, 8192, 8193])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_long_rows_of_more_tokens_than_compute_units(vecs, dt):
    """Vocabularies around the lengths at which a workgroup's threads hold more vectors of a row."""
    T = torch.cuda.get_device_properties(0).multi_processor_count + 5
    e = 4 if dt == "f32" else 8
    z, a, old, adv, ref, mask = _inputs(T, vecs * e + (vecs % 2) * 3, dt, 13)  # (odd ones: rows that end inside a vector)
    _check(z, a, old, adv, ref, mask, kl=0.1, scale=1024.0 if dt == "f16" else 1.0)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 1024, 33000])
def test_tokens_left_out(dt, V):
    """Masked rows hold NaN, infinities and an index that is none: nothing of it comes through."""
    z, a, old, adv, ref, mask = _inputs(24, V, dt, 3)
    mask[0], mask[5], mask[1] = False, False, True
    for t, v in ((z, math.nan), (old, math.inf), (adv, math.nan), (ref, -math.inf)):
        t[0] = v
    z[5] = -math.inf
    a[0], a[5] = -100, V + 7
    clean = [t.clone() for t in (z, a, old, adv, ref)]
    for t in clean:
        t[~mask] = 0
    kw = dict(kl_coef=0.1)
    got = policy_loss_and_grad(z, a, old, adv, ref, mask, **kw)
    want = policy_loss_and_grad(*clean, mask, **kw)
    assert all(torch.equal(p, q) for p, q in zip(got, want)) and got[0].isfinite()
    zz = z.requires_grad_(True)
    loss, _ = policy_loss(zz, a, old, adv, ref, mask, **kw)
    g, = torch.autograd.grad(loss, zz)
    assert g.isfinite().all() and not g[~mask].any()


@pytest.mark.parametrize("V", [40, 5000, 140000])
def test_exponentials_past_fp32_without_a_factor(V):
    """exp(lp - old) of a token without an advantage, and exp(ref - lp) with kl_coef 0, count for nothing when they overflow."""
    z, a, old, adv, ref, mask = _inputs(8, V, "f32", 12)
    mask[:4] = True
    z[torch.arange(2), a[:2]] = -150.0  # lp about -160, against a reference of about -8
    old[:2] = torch.log_softmax(z[:2].double(), 1).gather(1, a[:2, None])[:, 0].float() - 0.05
    old[2], adv[2] = -200.0, 0.0
    old[3], adv[3] = -200.0, 1.0  # held by the clip
    assert torch.exp(ref[0] + 150.0).isinf()
    _check(z, a, old, adv, ref, mask, kl=0.0)
    _check(z[2:], a[2:], old[2:], adv[2:], ref[2:], mask[2:], kl=0.1)


def test_nothing_counts():
    z, a, old, adv, ref, mask = _inputs(6, 50, "bf16", 4)
    z.requires_grad_(True)
    loss, logp = policy_loss(z, a, old, adv, ref, torch.zeros_like(mask))
    g, = torch.autograd.grad(loss, z)
    assert float(loss) == 0 and not logp.any() and not g.any()
    e = z.detach()[:0].requires_grad_(True)
    loss, logp = policy_loss(e, a[:0], old[:0], adv[:0], ref[:0], mask[:0])
    assert float(loss) == 0 and logp.shape == (0,)
    assert torch.autograd.grad(loss, e)[0].shape == (0, 50)
    loss, logp, g = policy_loss_and_grad(e.detach(), a[:0], old[:0], adv[:0])
    assert float(loss) == 0 and g.shape == (0, 50)


@pytest.mark.parametrize("V", [64, 5000])
def test_values_masked_by_infinity_and_the_lowest_number(V):
    z, a, old, adv, ref, mask = _inputs(12, V, "f32", 5)
    allowed = torch.rand(12, V, device="cuda") < 0.5
    allowed[torch.arange(12), a] = True
    for low in (-math.inf, torch.finfo(torch.float32).min):
        zz = torch.where(allowed, z, low)
        lp = torch.log_softmax(zz.double(), 1).gather(1, a[:, None])[:, 0].float()
        loss, logp, g = policy_loss_and_grad(zz, a, lp, adv, kl_coef=0.0)
        assert (logp - lp).abs().max() <= (V / 512 + 64 + 4 * 60) * U32
        assert g.isfinite().all() and not g[~allowed].any()
    only = torch.full((12, V), -math.inf, device="cuda")
    only[torch.arange(12), a] = 3.0  # one value allowed: probability 1, no gradient
    loss, logp, g = policy_loss_and_grad(only, a, torch.zeros(12, device="cuda"), adv)
    assert not logp.any() and not g.any()


def test_non_finite_tokens_show_and_stay_in_their_rows():
    z, a, old, adv, ref, _ = _inputs(10, 200, "bf16", 6)
    z[2, 5], a[4], a[6] = math.nan, 200, -1
    z[8] = -math.inf
    loss, logp, g = policy_loss_and_grad(z, a, old, adv, ref, denominator=10.0)
    bad = torch.zeros(10, dtype=torch.bool, device="cuda")
    bad[[2, 4, 6, 8]] = True
    assert loss.isnan() and logp[bad].isnan().all() and logp[~bad].isfinite().all()
    assert g[bad].isnan().any(1).all() and g[~bad].isfinite().all()
    keep = torch.nonzero(~bad)[:, 0]
    _, _, clean = policy_loss_and_grad(z[keep], a[keep], old[keep], adv[keep], ref[keep], denominator=10.0)
    assert torch.equal(g[keep], clean)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("V", [7, 64, 1001])
def test_strides_and_starts(dt, V):
    z, a, old, adv, ref, mask = _inputs(30, V, dt, 7)
    kw = dict(ref_logp=ref, mask=mask, kl_coef=0.2)
    want = policy_loss_and_grad(z, a, old, adv, **kw)

    def same(logits, a=a):
        got = policy_loss_and_grad(logits, a, old, adv, **kw)
        for p, q in zip(got, want):  # other vectors: another order of a row's sum
            assert (p.float() - q.float()).abs().max() <= 2.0 ** -7 * q.float().abs().max()
        zz = logits.detach().requires_grad_(True)
        g, = torch.autograd.grad(policy_loss(zz, a, old, adv, **kw)[0], zz)
        assert g.shape == zz.shape and (g.float() - want[2].float()).abs().max() <= 2.0 ** -7 * want[2].float().abs().max()

    wide = torch.full((30, V + 5), math.nan, dtype=z.dtype, device="cuda")
    for at in (0, 1, 5):
        part = wide[:, at:at + V]
        part.copy_(z)
        same(part)
        wide.fill_(math.nan)
    flat = torch.full((30 * V + 9,), math.nan, dtype=z.dtype, device="cuda")
    for at in (1, 3):
        same(flat[at:at + 30 * V].view(30, V).copy_(z))
    same(z.t().contiguous().t())
    same(z, a.int())
    b = policy_loss_and_grad(z.view(5, 6, V), a.view(5, 6), old.view(5, 6), adv.view(5, 6), ref.view(5, 6), mask.view(5, 6), kl_coef=0.2)
    assert torch.equal(b[2].view(30, V), want[2]) and b[1].shape == (5, 6) and torch.equal(b[0], want[0])


def test_against_differences():
    z, a, old, adv, ref, mask = _inputs(9, 40, "f32", 8)
    kw = dict(lo=0.2, hi=0.3, kl=0.3)
    _, _, g = policy_loss_and_grad(z, a, old, adv, ref, mask, 0.2, 0.3, 0.3)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(4):
        v, h = torch.randn(9, 40, generator=gen, device="cuda").double(), 1e-6
        up, down = (policy64(z.double() + s * h * v, a, old, adv, ref, mask, **kw)[0] for s in (1, -1))
        assert abs(float((g.double() * v).cpu().sum()) - float(up - down) / (2 * h)) <= 1e-5 * float((g.double() * v).abs().cpu().sum()) + 1e-8


def test_on_another_stream_in_a_graph_and_again():
    z, a, old, adv, ref, mask = _inputs(200, 5003, "bf16", 9)
    zz = z.requires_grad_(True)

    def step():
        loss, logp = policy_loss(zz, a, old, adv, ref, mask, kl_coef=0.1)
        g, = torch.autograd.grad(loss, zz)
        return (loss.detach(), logp, g, *policy_loss_and_grad(zz, a, old, adv, ref, mask, kl_coef=0.1))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            zz.add_(torch.randn_like(zz))
            for t in held:
                t.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step())), k


def test_timer_and_second_derivatives():
    z, a, old, adv, ref, mask = _inputs(20, 100, "f32", 10)
    zz = z.requires_grad_(True)
    want, = torch.autograd.grad(policy_loss(zz, a, old, adv)[0], zz)
    with kernel_timer() as kt:
        got, = torch.autograd.grad(policy_loss(zz, a, old, adv)[0], zz)
        policy_loss_and_grad(zz, a, old, adv)
    assert set(kt.stats()) == {"policy_loss_fwd", "policy_loss_bwd", "policy_loss_and_grad"} and torch.equal(got, want)
    g, = torch.autograd.grad(policy_loss(zz, a, old, adv)[0], zz, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.square().sum().backward()


def test_more_than_2_31_logits():
    T, V = 33000, 65536 + 8
    z = torch.zeros(T, V, dtype=torch.bfloat16, device="cuda")
    a = torch.full((T,), V - 1, device="cuda")
    z[:, V - 1] = 8.0
    old, adv = torch.full((T,), -5.0, device="cuda"), torch.ones(T, device="cuda")
    z[-50:, :1000] = 1.0
    loss, logp, g = policy_loss_and_grad(z, a, old, adv, denominator=1.0, clip_high=100.0)
    assert torch.equal(logp[:T - 50], logp[:1].expand(T - 50))
    _, want_lp, want = policy_loss_and_grad(z[-60:].clone(), a[-60:], old[-60:], adv[-60:], denominator=1.0, clip_high=100.0)
    assert torch.equal(g[-60:], want) and torch.equal(logp[-60:], want_lp)


def test_refusals():
    z, a, old, adv, ref, mask = _inputs(6, 50, "bf16", 11)
    good = dict(logits=z, actions=a, old_logp=old, advantages=adv, ref_logp=ref, mask=mask)
    for bad in [dict(logits=z.cpu()), dict(actions=a.cpu()), dict(actions=a.float()), dict(actions=a[:-1]), dict(old_logp=old[:, None]),
                dict(advantages=adv[:-1]), dict(ref_logp=ref.long()), dict(mask=mask.long()), dict(mask=mask[:-1]), dict(logits=z.double()),
                dict(logits=z[:, :0]), dict(clip_low=-0.1), dict(clip_high=math.nan), dict(denominator=0.0), dict(denominator=-1.0)]:
        for fn in (policy_loss, policy_loss_and_grad):
            with pytest.raises(ValueError):
                fn(**(good | bad))
