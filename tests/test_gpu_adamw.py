"""GPU parity of adamw_step_hip / AdamW: bitwise with the elementary form, and with the formula in float64."""

import math

import pytest
import torch

from tests._train import LEAST, U32, UNIT, close

from mhc_mlx_amd import AdamW, MHCLayer, adamw_step_hip, kernel_timer
from mhc_mlx_amd.optim import BLOCK, _decode, _encode, adamw_step_reference

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(step=7, lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _lists(shapes, dt, bits=32, master=False, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)

    def normal(shape, scale):
        return torch.randn(*shape, generator=g) * scale

    out = {k: [] for k in ("params", "grads", "exp_avgs", "exp_avg_sqs", "masters", "scales")}
    for i, shape in enumerate(shapes):
        w = normal(shape, 0.5)
        m, v = normal(shape, 0.01), normal(shape, 0.02).square()
        out["params"].append(w.to(DT[dt]))
        out["grads"].append(normal(shape, 0.02).to(DT[dt]))
        out["masters"].append(w if master else None)
        if bits == 8:
            (m, mu), (v, vu) = _encode(m.reshape(-1)), _encode(v.sqrt().reshape(-1))
            out["scales"].append(torch.stack([mu, vu], 1))
            m, v = m.view(w.shape), v.view(w.shape)
        out["exp_avgs"].append(m)
        out["exp_avg_sqs"].append(v)
    out["masters"] = out["masters"] if master else None
    out["scales"] = out["scales"] if bits == 8 else None
    return {k: None if v is None else [t.to(device) for t in v] for k, v in out.items()}


def _clone(lists, device=None):
    return {k: None if v is None else [t.clone().to(device or t.device) for t in v] for k, v in lists.items()}


def _bits(t):
    return t.contiguous().view(torch.uint8) if t.numel() else t


def _same(a, b):
    for k in a:
        for i, (s, t) in enumerate(zip(a[k] or [], b[k] or [])):
            assert torch.equal(_bits(s.cpu()), _bits(t.cpu())), (k, i)


SHAPES = [(1,), (4,), (4, 4), (3,), (255,), (256,), (257,), (1024,), (1000, 3), (4096,), (4097,), (77, 129), (0,), (5, 0, 2), (16384,)]


@pytest.mark.parametrize("dt,master", [("f32", False), ("bf16", False), ("bf16", True), ("f16", False), ("f16", True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_bitwise_with_the_elementary_form(dt, master, bits):
    """Three steps on the GPU and, in elementary operations, on the CPU."""
    a = _lists(SHAPES, dt, bits, master)
    b = _clone(a, "cpu")
    for k in range(3):
        adamw_step_hip(**a, **(HYPER | dict(step=7 + k)))
        adamw_step_reference(**b, **(HYPER | dict(step=7 + k)))
    _same(a, b)


@pytest.mark.parametrize("dt,master", [("f32", False), ("bf16", True), ("f16", False)])
def test_formula_in_64_bits(dt, master):
    a = _lists([(3000,), (33, 65)], dt, 32, master, 1)
    start = _clone(a)
    adamw_step_hip(**a, **HYPER)
    t, lr, (b1, b2), eps, wd = (HYPER[k] for k in ("step", "lr", "betas", "eps", "weight_decay"))
    for i in range(2):
        p = (start["masters"] if master else start["params"])[i].double()
        g, m, v = (start[k][i].double() for k in ("grads", "exp_avgs", "exp_avg_sqs"))
        m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        update = lr / (1 - b1 ** t) * m1 / (torch.sqrt(v1 / (1 - b2 ** t)) + eps)
        p1 = p - lr * wd * p - update
        m_off = 4 * U32 * (b1 * m.abs() + (1 - b1) * g.abs())
        v_off = 6 * U32 * v1 + 2.0 ** -149
        close(a["exp_avgs"][i], m1, m_off, "m")
        close(a["exp_avg_sqs"][i], v1, v_off, "v")
        # m's roundings count as they are, v's by half, then some ten of the step's own
        size = lr / (1 - b1 ** t) / (torch.sqrt(v1 / (1 - b2 ** t)) + eps)
        off = size * m_off + 16 * U32 * update.abs() + 3 * U32 * p.abs()
        if master:
            close(a["masters"][i], p1, off, "master")
            assert torch.equal(a["params"][i], a["masters"][i].to(DT[dt]))
        close(a["params"][i], p1, off * 1.01 + UNIT[DT[dt]] * 1.01 * p1.abs() + LEAST[DT[dt]], "p")


def test_codes_hold_what_they_stand_for():
    a = _lists([(4096 + 100,)], "f32", 8, False, 2)
    start = _clone(a)
    adamw_step_hip(**a, **HYPER)
    g = start["grads"][0].double()
    m = _decode(start["exp_avgs"][0], start["scales"][0][:, 0]).double()
    r = _decode(start["exp_avg_sqs"][0], start["scales"][0][:, 1]).double()
    for want, codes, unit in ((0.9 * m + 0.1 * g, a["exp_avgs"][0], a["scales"][0][:, 0]),
                              (torch.sqrt(0.95 * r * r + 0.05 * g * g), a["exp_avg_sqs"][0], a["scales"][0][:, 1])):
        got, u = _decode(codes, unit).double(), unit.double().repeat_interleave(BLOCK)[:want.numel()]
        # half of the last of three bits: 2^-4 of the value, or 2^-10 units below the least normal code
        close(got, want, (2.0 ** -4 + 1e-5) * want.abs() + (2.0 ** -10) * u, "state")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("by", [1, 2, 3, 5])
def test_starts_and_holes(bits, by):
    """Tensors that start off a vector, next to memory that must not change."""
    a = _lists([(1001,), (7,), (513,)], "bf16", bits, True, 3)
    b = _clone(a)
    for k, v in a.items():
        if v is None or k == "scales":
            continue
        for i, t in enumerate(v):
            flat = torch.full((t.numel() + by + 9,), 0x3c, dtype=torch.uint8, device="cuda") if t.element_size() == 1 else \
                torch.full((t.numel() + by + 9,), 3.0, dtype=t.dtype, device="cuda")
            flat = flat.view(t.dtype)
            flat[by:by + t.numel()].copy_(t)
            v[i] = flat[by:by + t.numel()]
    adamw_step_hip(**a, **HYPER)
    adamw_step_hip(**b, **HYPER)
    _same(a, b)
    for v in (a["params"], a["masters"], a["exp_avgs"], a["exp_avg_sqs"]):
        for t in v:
            whole = t._base if t._base is not None else t
            whole = whole.view(t.dtype)
            edge = torch.cat([_bits(whole[:by]), _bits(whole[by + t.numel():])])
            one = _bits(torch.full((1,), 3.0, device="cuda").to(t.dtype)) if t.element_size() > 1 else torch.tensor([0x3c], dtype=torch.uint8, device="cuda")
            assert torch.equal(edge, one.repeat(by + 9))


def test_orders_of_axes():
    """A parameter in another order of its axes, its gradient in a third."""
    w = torch.randn(12, 20, 6, device="cuda")
    args = dict(exp_avgs=[torch.zeros_like(w)], exp_avg_sqs=[torch.zeros_like(w)])
    p = w.permute(2, 0, 1)
    other = [p.clone(), p.contiguous()]
    g = torch.randn(6, 12, 20, device="cuda")
    adamw_step_hip([p], [g], [args["exp_avgs"][0].permute(2, 0, 1)], [args["exp_avg_sqs"][0].permute(2, 0, 1)], **HYPER)
    adamw_step_hip([other[1]], [g], [torch.zeros_like(other[1])], [torch.zeros_like(other[1])], **HYPER)
    assert torch.equal(p, other[1]) and not torch.equal(p, other[0])


@pytest.mark.parametrize("count", [59, 60, 61, 130])
def test_many_tensors_and_dtypes_in_one_call(count):
    lists = [_lists([(4,), (16,), (1025,)] * count, d, 32, False, 5) for d in ("f32", "bf16")]
    a = {k: None if lists[0][k] is None else [t for pair in zip(lists[0][k], lists[1][k]) for t in pair] for k in lists[0]}
    b = _clone(a, "cpu")
    adamw_step_hip(**a, **HYPER)
    adamw_step_reference(**b, **HYPER)
    _same(a, b)


def test_gradient_scale():
    a = _lists([(1000,), (9,)], "f32", 32, False, 6)
    b, c, d = _clone(a), _clone(a), _clone(a)
    adamw_step_hip(**a, **HYPER, grad_scale=0.3)
    adamw_step_hip(**b, **HYPER, grad_scale=torch.tensor(0.3, device="cuda"))
    _same(a, b)
    c["grads"] = [g * 0.3 for g in c["grads"]]
    adamw_step_hip(**c, **HYPER)
    for k in ("params", "exp_avgs", "exp_avg_sqs"):
        assert all(torch.equal(s, t) for s, t in zip(a[k], c[k]))
    adamw_step_hip(**d, **HYPER, grad_scale=torch.tensor([0.3], device="cuda"))
    _same(a, d)


@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_and_extreme_gradients(bits):
    a = _lists([(1024,)], "f32", bits, False, 7)
    g = a["grads"][0]
    g[3], g[300], g[600], g[601], g[1000] = math.nan, math.inf, 1e-30, 1e30, 0.0
    b = _clone(a, "cpu")
    adamw_step_hip(**a, **HYPER)
    adamw_step_reference(**b, **HYPER)
    for k in ("params", "exp_avgs", "exp_avg_sqs") + (("scales",) if bits == 8 else ()):
        s, t = a[k][0].cpu().float(), b[k][0].float()
        assert torch.equal(s.isnan(), t.isnan()) and torch.equal(s.nan_to_num(0.5), t.nan_to_num(0.5)), k
    assert a["params"][0][768:].isfinite().all() and a["params"][0][4:256].isfinite().all()
    zero = _lists([(512,)], "f32", bits, False, 8)
    for k in ("grads", "exp_avgs", "exp_avg_sqs"):
        zero[k][0].view(torch.uint8).zero_()
    if bits == 8:
        zero["scales"][0].zero_()
    before = zero["params"][0].clone()
    adamw_step_hip(**zero, **HYPER)
    assert torch.equal(zero["params"][0], before * (1.0 - HYPER["lr"] * HYPER["weight_decay"]))
    assert not zero["exp_avgs"][0].float().any() and all(t[0].float().isfinite().all() for t in zero.values() if t)


def test_saved_tensors_notice_the_step():
    a = _lists([(32,)], "f32")
    w = a["params"][0].requires_grad_(True)
    y = (w * w).sum()
    with torch.no_grad():
        adamw_step_hip(**a, **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_on_another_stream_and_in_a_graph():
    a = _lists([(5000,), (4,)] * 40, "bf16", 8, True, 9)
    b, c = _clone(a), _clone(a)
    adamw_step_hip(**a, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adamw_step_hip(**b, **HYPER)
    torch.cuda.current_stream().wait_stream(side)
    _same(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adamw_step_hip(**c, **HYPER)
    graph.replay()
    torch.cuda.synchronize()
    _same(a, c)
    for _ in range(2):
        for g, h in zip(a["grads"], c["grads"]):
            g.mul_(-0.5)
            h.mul_(-0.5)
        adamw_step_hip(**a, **HYPER)
        graph.replay()
        torch.cuda.synchronize()
        _same(a, c)


def test_more_than_2_31_elements():
    n = 2 ** 31 + 4099
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    s = torch.zeros(-(-n // 256), 2, device="cuda")
    g[-5000:] = 0.25
    adamw_step_hip([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0, scales=[s])
    assert bool((p[-5000:] == -0.5).all()) and not p[:-5000:1013].any() and not p[-6000:-5000].any()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_optimizer_on_the_gpu_is_the_one_on_the_cpu(bits, dt):
    torch.manual_seed(0)
    ws = [torch.randn(s).to(DT[dt]) for s in ((70, 90), (5,), (64, 64), (3, 3))]
    sides = []
    for device in ("cuda", "cpu"):
        ps = [torch.nn.Parameter(w.clone().to(device)) for w in ws]
        sides.append((ps, AdamW([dict(params=ps[:2]), dict(params=ps[2:], weight_decay=0.0, lr=3e-3)], state_bits=bits)))
    for k in range(4):
        for ps, opt in sides:
            gen = torch.Generator().manual_seed(k)
            for i, p in enumerate(ps):
                grad = torch.randn(p.shape, generator=gen)
                p.grad = None if i == 1 and k == 1 else grad.to(p.device, p.dtype)
            opt.step(grad_scale=0.5)
        if k == 2:  # saved and loaded on the way
            ps, opt = sides[0]
            fresh = AdamW([dict(params=ps[:2]), dict(params=ps[2:])], state_bits=bits)
            fresh.load_state_dict(opt.state_dict())
            sides[0] = (ps, fresh)
    for p, q in zip(sides[0][0], sides[1][0]):
        assert torch.equal(p.cpu(), q)
        s, t = sides[0][1].state[p], sides[1][1].state[q]
        assert s["step"] == t["step"] and set(s) == set(t)
        assert all(torch.equal(_bits(s[k].cpu()), _bits(t[k])) for k in s if k != "step")


def test_trains_an_mhc_layer():
    torch.manual_seed(0)
    layer = MHCLayer(4, 64, identity_init=False).cuda()
    x, want = torch.randn(256, 4, 64, device="cuda"), torch.randn(256, 4, 64, device="cuda")
    opt = AdamW(layer.parameters(), lr=0.05, weight_decay=0.0)
    losses = []
    for _ in range(12):
        opt.zero_grad()
        loss = (layer(x) - want).square().mean()
        loss.backward()
        opt.step()
        losses.append(float(loss))
    assert losses[-1] < 0.95 * losses[0]
    with kernel_timer() as kt:
        opt.step()
    assert "adamw_step" in kt.stats()


def test_refusals():
    def step(**change):
        a = _lists([(300,), (4,)], change.pop("dt", "bf16"), change.pop("bits", 32), change.pop("master", True))
        numbers = dict(HYPER)
        for k, v in change.items():
            if k in a:
                a[k] = v(a[k])
            else:
                numbers[k] = v
        adamw_step_hip(**a, **numbers)

    step()
    step(bits=8)
    first = lambda f: lambda ts: [f(ts[0]), *ts[1:]]  # noqa: E731
    for bad in [dict(params=lambda t: t[:1]), dict(grads=lambda t: t[:1]), dict(masters=lambda t: t[:1]), dict(params=first(lambda t: t.cpu())),
                dict(grads=first(lambda t: t.cpu())), dict(grads=first(lambda t: t.float())), dict(grads=first(lambda t: t[:-1])),
                dict(exp_avgs=first(lambda t: t.half())), dict(exp_avg_sqs=first(lambda t: t[:-1])), dict(masters=first(lambda t: t.half())),
                dict(dt="f32"), dict(params=first(lambda t: t.double())), dict(params=first(lambda t: t[:1].expand(300))),
                dict(grads=first(lambda t: t.to_sparse())), dict(bits=8, scales=first(lambda t: t[:-1])), dict(bits=8, scales=lambda t: None),
                dict(bits=8, scales=lambda t: t[:1]), dict(step=0), dict(step=1.5), dict(lr=-1.0), dict(lr=math.nan), dict(betas=(0.9, 1.0)),
                dict(betas=(0.9,)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(grad_scale=torch.tensor(1.0)),
                dict(grad_scale=torch.ones(2, device="cuda")), dict(grad_scale=torch.ones(1, device="cuda").double())]:
        with pytest.raises(ValueError):
            step(**bad)
    adamw_step_hip([], [], [], [], step=1)


@pytest.mark.parametrize("count", [63, 64, 65, 72, 73, 84, 85, 100, 101, 128, 129, 201])
@pytest.mark.parametrize("dt,bits,master", [("f32", 32, False), ("f32", 8, False), ("bf16", 32, True), ("f16", 8, True)])
def test_lists_around_the_length_of_a_launch(count, dt, bits, master):
    """Tensors of one and of several workgroups, in numbers at which a launch's table or a vote ends."""
    shapes = [((5, 1024, 1025, 300, 2048)[i % 5],) for i in range(count)]
    a = _lists(shapes, dt, bits, master, 7)
    b = _clone(a, "cpu")
    adamw_step_hip(**a, **HYPER)
    adamw_step_reference(**b, **HYPER)
    _same(a, b)
