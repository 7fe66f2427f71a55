"""add_rms_norm, its int8 form and quantize_int8 on the GPU against float64 (tests/_block.py)."""

import pytest
import torch

from mhc_mlx_amd import AddRMSNorm, add_rms_norm, add_rms_norm_int8, kernel_timer, quantize_int8
from tests._block import check_codes, norm64, norm_grads64, normed64, ones
from tests._train import U32, close

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6
# one element to rows that no workgroup holds; widths off every vector's length, and around what each kernel holds
WIDTHS = [1, 7, 64, 65, 250, 512, 1100, 2047, 2050, 4096, 5001, 8192, 16384, 16392, 40000, 70001]


def rand(g, *shape, dt=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(seed, T, C, dt, residual=True, weight="same"):
    g = gen(seed)
    x, r = rand(g, T, C, dt=dt), rand(g, T, C, dt=dt, scale=2.0) if residual else None
    w = None if weight is None else (1 + 0.3 * rand(g, C)).to(torch.float32 if weight == "fp32" else dt)
    return x, r, w


def check_all(x, r, w, seed, with_dh=True):
    """Forward and gradients of one call."""
    g = gen(seed + 1000)
    T, C = x.shape
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, r, w)]
    y, h = add_rms_norm(*leaves, eps=EPS)
    h0, y0, bound = normed64(x, r, w, EPS)
    assert torch.equal(h, h0) and y.dtype == x.dtype
    close(y, y0, bound, "y")
    dy, dh = rand(g, T, C, dt=x.dtype), rand(g, T, C, dt=x.dtype) if r is not None and with_dh else None
    given = [t for t in leaves if t is not None]
    outs, ups = ([y, h], [dy, dh]) if dh is not None else ([y], [dy])
    grads = torch.autograd.grad(outs, given, ups)
    _, z, s, off = norm64(x, r, w, EPS)
    (dx, bdx), (dw, bdw) = norm_grads64(h0, z, s, off, w, dy, dh, x.dtype, x.dtype if w is None else w.dtype)
    close(grads[0], dx, bdx, "dx")
    if r is not None:
        assert torch.equal(grads[0], grads[1])
    if w is not None:
        close(grads[-1], dw, bdw, "dw")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_forward_and_gradients(dt, C):
    for k, (T, residual, weight) in enumerate([(1, True, "same"), (3, False, "fp32"), (70, True, "fp32"), (5, True, None), (2, False, None)]):
        x, r, w = inputs(C + k, T, C, dt, residual, weight)
        check_all(x, r, w, C + k, with_dh=k != 3)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,C", [(4097, 64), (1500, 1100), (3000, 2048), (1027, 8200)])
def test_many_rows(dt, T, C):
    check_all(*inputs(T, T, C, dt, True, "fp32"), seed=T)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_int8(dt, C):
    for k, (T, residual, weight) in enumerate([(1, True, "same"), (6, False, "fp32"), (33, True, None)]):
        x, r, w = inputs(C + k + 7, T, C, dt, residual, weight)
        rows, h = add_rms_norm_int8(x, r, w, eps=EPS)
        h0, z, s, off = norm64(x, r, w, EPS)
        assert torch.equal(h, h0) and rows.codes.dtype == torch.int8 and rows.scales.shape == (T,)
        v = z * s * ones(w, z)
        check_codes(rows.codes, rows.scales, v, off)
        if dt == torch.bfloat16 and weight != "fp32":  # every product is exact, and so is each code
            p = z * ones(w, z)
            assert torch.equal(rows.codes.double(), torch.round(127 * p / p.abs().amax(1, keepdim=True)))
        q = quantize_int8(x)
        check_codes(q.codes, q.scales, x.double(), 0.0)


@pytest.mark.parametrize("T,C", [((1 << 22) + 7, 6), ((1 << 20) + 9, 2056)])
def test_more_rows_than_a_launch_has_workgroups(T, C):
    """Rows that go round again: first, middle and last ones against float64, and every scale."""
    g = gen(T)
    x = torch.empty(T, C, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    w = (1 + 0.3 * rand(g, C)).bfloat16()
    at = torch.tensor([0, 1, 255, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, T - 2, T - 1], device="cuda")
    y, _ = add_rms_norm(x, None, w, eps=EPS)
    _, y0, bound = normed64(x[at], None, w, EPS)
    close(y[at], y0, bound, "y")
    del y
    q = quantize_int8(x)
    check_codes(q.codes[at], q.scales[at], x[at].double(), 0.0)
    assert torch.allclose(q.scales, x.abs().amax(1).float() / 127, rtol=1e-6, atol=0)
    del q
    if C > 6:
        return
    xs, ws = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(add_rms_norm(xs, None, ws, eps=EPS)[0], [xs, ws], torch.ones_like(x))
    h, z, s, off = norm64(x, None, w, EPS)
    (rdx, bdx), (rdw, bdw) = norm_grads64(h, z, s, off, w, torch.ones_like(x), None, x.dtype, w.dtype)
    close(dx, rdx, bdx, "dx")
    close(dw, rdw, bdw, "dw")


def test_codes_of_ties_and_of_extreme_values():
    """Halves go to the even code, and the largest and smallest values of fp32 have their codes."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5]], device="cuda")
    want = torch.tensor([[127, 0, 2, 2, 0, -2, -126, 126]], dtype=torch.int8, device="cuda")
    for dt in DTYPES:
        q = quantize_int8(x.to(dt))
        assert torch.equal(q.codes, want) and float(q.scales) == 1.0
    for k in (-149 + 20, -126, -100, 60, 120):  # (times a power of two: the same codes, also where the values are subnormal)
        big = x.double() * 2.0 ** k
        fits = big.float().double() == big
        got = quantize_int8(big.float())
        assert torch.equal(got.codes[fits], want[fits])
    m = torch.finfo(torch.float32).max
    assert quantize_int8(torch.tensor([[m, -m, m / 2, 0.0]], device="cuda")).codes.tolist() == [[127, -127, 64, 0]]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("C", [5, 64, 3000, 40000])
def test_rows_of_zeros_and_of_infinities(dt, C):
    x = rand(gen(C), 4, C, dt=dt)
    x[1] = 0
    x[2, C // 2] = float("inf")
    x[3, C - 1] = float("nan")
    w = torch.ones(C, device="cuda", dtype=dt)
    for rows in (quantize_int8(x), add_rms_norm_int8(x, None, w)[0]):
        assert rows.scales[1] == 0 and not rows.codes[1].any()
        assert bool(rows.scales[2:].isnan().all()) and not rows.codes[2:].any()
        assert bool(rows.scales[0] > 0)
    x.requires_grad_(True)
    y, _ = add_rms_norm(x, None, w)
    assert not y[1].any() and bool(y[3].isnan().all()) and bool(y[2, C // 2].isnan())
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool(dx[:2].isfinite().all()) and bool(dx[3].isnan().all())
    # a weight that is not finite
    w[0] = float("inf")
    rows, _ = add_rms_norm_int8(x.detach(), None, w)
    assert bool(rows.scales[0].isnan()) and not rows.codes[0].any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [48, 1024, 9000, 50000])
def test_squares_past_the_range(dt, C):
    """Values whose squares' sum is past fp32's range are normed all the same."""
    for scale in (1e19, 1e30, 3e37):
        x = rand(gen(C), 3, C, dt=dt).clamp(-4, 4) * scale
        x[1] = 1.0  # (a row beside them is not touched)
        h, y, bound = normed64(x, None, None, EPS)
        # (the factor may be a subnormal number: its last bit is then 2^-150 of 1 / scale)
        close(add_rms_norm(x, eps=EPS)[0], y, bound + (4 * U32 + 2.0 ** -149 * scale * 4) * y.abs(), f"{scale}")
        rows, _ = add_rms_norm_int8(x, eps=EPS)
        z = h.double()
        check_codes(rows.codes, rows.scales, y, (C + 8) * U32 + 2.0 ** -149 * scale * 4)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [48, 1024, 9000, 50000])
def test_codes_of_products_past_the_range(dt, C):
    """Rows up to 1.2e38 times weights around 20: the products are past fp32's range, the normed values are around 20."""
    x = rand(gen(C), 3, C, dt=dt).clamp(-4, 4) * 3e37
    x[1] = 1.0  # (a row beside them is not touched)
    w = (20 * (1 + 0.3 * rand(gen(C + 1), C))).to(dt)
    h, z, s, _ = norm64(x, None, w, EPS)
    rows, _ = add_rms_norm_int8(x, None, w, eps=EPS)
    # (eps is nothing beside those squares)
    check_codes(rows.codes, rows.scales, z * s * ones(w, z), (C + 8) * U32)


def test_strides_and_shapes():
    g = gen(3)
    wide = rand(g, 6, 5, 300, dt=torch.bfloat16)
    for x in (wide[:, :, 3:131], wide[::2, 1, 10:138], wide.transpose(0, 1)[..., :128], wide[:, :, ::2][..., :128], wide[0, 0, :128],
              wide[:1, :1, 5:133].expand(4, 3, 128)):
        r = rand(g, *x.shape, dt=torch.bfloat16)
        w = rand(g, 128, 2, dt=torch.float32)[:, 1]
        y, h = add_rms_norm(x, r, w)
        want, hw = add_rms_norm(x.contiguous(), r, w.contiguous())
        assert y.shape == x.shape and torch.equal(y, want) and torch.equal(h, hw)
        a, _ = add_rms_norm_int8(r, x, w)
        b, _ = add_rms_norm_int8(r, x.contiguous(), w.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.scales.shape == x.shape[:-1]
        q, k = quantize_int8(x), quantize_int8(x.contiguous())
        assert torch.equal(q.codes, k.codes) and torch.equal(q.scales, k.scales)
    # gradients that come in other layouts
    x = rand(g, 6, 40).requires_grad_(True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    y, _ = add_rms_norm(x, None, w)
    up = rand(g, 40, 6).t()
    a = torch.autograd.grad(y, [x, w], up, retain_graph=True)
    b = torch.autograd.grad(y, [x, w], up.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y, _ = add_rms_norm(x, None, w)
    y.sum().backward()  # (an expanded gradient)
    assert torch.equal(w.grad, torch.autograd.grad(add_rms_norm(x, None, w)[0], w, torch.ones(6, 40, device="cuda"))[0])


def test_no_rows():
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, h = add_rms_norm(x, x, w)
    assert y.shape == h.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16) and not w.grad.any()
    rows, _ = add_rms_norm_int8(x, None, w)
    assert rows.codes.shape == (0, 16) and rows.scales.shape == (0,) and quantize_int8(x).codes.shape == (0, 16)


def test_which_gradients_are_asked_for():
    g = gen(8)
    x, r, w = rand(g, 9, 72), rand(g, 9, 72), rand(g, 72)
    ts = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, h = add_rms_norm(*ts)
    dy, dh = rand(g, 9, 72), rand(g, 9, 72)
    full = torch.autograd.grad([y, h], ts, [dy, dh], retain_graph=True)
    only_h = torch.autograd.grad(h, ts, dh, retain_graph=True, allow_unused=True)
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[1], dh) and not only_h[2].any()
    only_y = torch.autograd.grad(y, ts, dy)
    assert torch.equal(only_y[2], full[2])
    for k in range(3):
        one = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, r, w))]
        y, h = add_rms_norm(*one)
        d, = torch.autograd.grad([y, h], [one[k]], [dy, dh]) if k < 2 else torch.autograd.grad(y, [one[k]], dy)
        assert torch.equal(d, full[k])
    with torch.no_grad():
        y2, h2 = add_rms_norm(*ts)
    assert not y2.requires_grad and torch.equal(y2, y)
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        a = ts[0].detach().requires_grad_(True)
        d, = torch.autograd.grad(add_rms_norm(a)[0].sum(), a, create_graph=True)
        d.sum().backward()
    with kernel_timer() as kt:  # the Function in Python
        ts = [t.clone().requires_grad_(True) for t in (x, r, w)]
        y, h = add_rms_norm(*ts)
        timed = torch.autograd.grad([y, h], ts, [dy, dh])
        alone, _ = add_rms_norm(ts[0], None, ts[2])
        torch.autograd.grad(alone, [ts[0], ts[2]], dy)
    assert all(torch.equal(a, b) for a, b in zip(timed, full)) and kt.stats()["add_rms_norm_bwd"]["count"] == 2


def test_module_and_refusals():
    g = gen(9)
    m = AddRMSNorm(96, device="cuda")
    x = rand(g, 4, 96, dt=torch.bfloat16)
    assert torch.equal(m(x, x)[0], add_rms_norm(x, x, m.weight)[0])
    m8 = AddRMSNorm(96, int8=True, device="cuda", dtype=torch.bfloat16)
    rows, h = m8(x)
    assert torch.equal(rows.codes, quantize_int8(x).codes) and h is not None
    mixed = AddRMSNorm(96, device="cuda")(x, x.float())
    assert all(a.dtype == torch.float32 and torch.equal(a, b) for a, b in zip(mixed, add_rms_norm(x.float(), x.float(), m.weight)))
    half = AddRMSNorm(96, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        half.weight.copy_(rand(g, 96))
    y, h = half(x, x.float())  # (the sum has float32, the weight neither that nor the rows' dtype of before)
    assert torch.equal(y, add_rms_norm(h, None, half.weight.float())[0]) and h.dtype == torch.float32
    d, = torch.autograd.grad(y, half.weight, torch.ones_like(y))
    assert d.dtype == torch.bfloat16 and bool(d.isfinite().all())
    for bad in (dict(residual=x[:2]), dict(residual=x.float()), dict(weight=torch.ones(95, device="cuda")), dict(eps=0.0), dict(eps=float("nan")),
                dict(weight=torch.ones(96, device="cuda", dtype=torch.float16)), dict(weight=torch.ones(96)), dict(residual=x.cpu())):
        with pytest.raises(ValueError):
            add_rms_norm(x, **bad)
        with pytest.raises(ValueError):
            add_rms_norm_int8(x, **bad)
    for bad in (x.double(), x.cpu(), torch.ones(3, 0, device="cuda"), torch.ones(3, 8, device="cuda", dtype=torch.int32)):
        with pytest.raises(ValueError):
            quantize_int8(bad)


@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_run_the_kernels_again(grad):
    """torch.jit.trace keeps the calls as nodes, those without a gradient too."""
    from mhc_mlx_amd import Int8Linear, linear_cross_entropy_and_grad

    g = gen(12)
    targets = torch.randint(0, 50, (6,), generator=g, device="cuda")

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.lin = AddRMSNorm(64, device="cuda"), Int8Linear.from_linear(torch.nn.Linear(64, 32, device="cuda"))
            self.register_buffer("head", torch.randn(50, 64, generator=g, device="cuda"))

        def forward(self, x, r):
            y, h = self.norm(x, r)
            rows, _ = add_rms_norm_int8(x, r, self.norm.weight)
            loss, logp, dx, dw = linear_cross_entropy_and_grad(y.detach(), self.head, targets)
            return y, h, self.lin(rows), self.lin(x), rows.dequantize(torch.bfloat16), quantize_int8(h).scales, loss, logp, dx, dw

    f = Block()
    traced = torch.jit.trace(f, (rand(g, 6, 64).requires_grad_(grad), rand(g, 6, 64)), check_trace=False)
    for _ in range(2):
        x, r = rand(g, 6, 64).requires_grad_(grad), rand(g, 6, 64)
        with torch.set_grad_enabled(grad):
            got, want = traced(x, r), f(x, r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        if grad:
            up = rand(g, 6, 64)
            assert torch.equal(*(torch.autograd.grad(o[0], x, up)[0] for o in (got, want)))


def test_captured_calls_and_other_streams():
    """Forward, backward and int8 in one graph, replayed with other data and eager work between; the same on a stream of one's own."""
    g = gen(10)
    x, r, w, dy, dh = (rand(g, 65, 1024, dt=torch.bfloat16) for _ in range(5))
    w = w[0].clone()
    ops = torch.empty_like(x)

    def step():
        ts = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, h = add_rms_norm(*ts)
        rows, _ = add_rms_norm_int8(x, r, w)
        return [y.detach(), h.detach(), rows.codes, rows.scales, *torch.autograd.grad([y, h], ts, [dy, dh])]

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
    for k in range(3):
        for t in (x, r, dy, dh):
            t.copy_(rand(g, 65, 1024))
        ops.copy_(x).mul_(2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), k
