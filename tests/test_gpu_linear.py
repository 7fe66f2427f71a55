"""GPU parity of linear_act / FusedLinear with the formula in float64, within element-wise bounds (tests/_train.py)."""

import pytest
import torch

from tests._train import act64, close, linear64, linear_grads64

from mhc_mlx_amd import AutoPatcher, FusedLinear, MHCRewire, kernel_timer, linear_act
from mhc_mlx_amd.linear import ACTIVATIONS, linear_act_reference

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(M, N, K, dt, seed=0, bias=True, residual=True, out=None):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + N * 3 + K)

    def normal(*shape, scale=1.0, dtype=DT[dt]):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    return (normal(M, K), normal(N, K, scale=K ** -0.5), normal(N) if bias else None,
            normal(M, N, dtype=out or DT[dt]) if residual else None, normal(M, N, scale=0.3, dtype=out or DT[dt]))


def _check(x, w, b, r, g, act, out_dtype=None):
    """Output and all gradients of 2-d inputs within their bounds."""
    ts = [t for t in (x, w, b, r) if t is not None]
    for t in ts:
        t.requires_grad_(True)
    out = linear_act(x, w, b, r, activation=act, output_dtype=out_dtype)
    want = out_dtype or x.dtype
    assert out.dtype == want
    ref, bound, _, d, dz = linear64(x, w, b, r, act, want)
    close(out, ref, bound, "out")
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, r, activation=act, output_dtype=out_dtype), out)
    grads = dict(zip("xwbr"[:2] + ("b" if b is not None else "") + ("r" if r is not None else ""), torch.autograd.grad(out, ts, g)))
    dx, dw, db = linear_grads64(x, w, g, d, dz, x.dtype, act != "none")
    close(grads["x"], *dx, "dx")
    close(grads["w"], *dw, "dw")
    if b is not None:
        close(grads["b"], *db, "db")
    if r is not None:
        assert torch.equal(grads["r"], g)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 256, 512), (2, 100, 60), (5, 33, 1000), (16, 512, 256), (17, 64, 96), (31, 129, 257),
                                   (64, 320, 192), (65, 1000, 72), (127, 384, 640), (128, 128, 64), (130, 257, 129), (257, 96, 2048),
                                   (300, 1100, 520), (513, 768, 256), (1000, 50, 33)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_sizes(M, N, K, dt):
    _check(*_inputs(M, N, K, dt), "gelu")


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("dt,out", [("f32", None), ("bf16", None), ("f16", None), ("bf16", torch.float32), ("f16", torch.float32)])
@pytest.mark.parametrize("M", [3, 200])
def test_activations_and_output_dtypes(act, dt, out, M):
    _check(*_inputs(M, 136, 264, dt, 1, out=out), act, out)


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("M", [4, 96])
def test_without_bias_or_residual(act, bias, residual, M):
    _check(*_inputs(M, 130, 96, "bf16", 2, bias, residual), act)


@pytest.mark.parametrize("M,N,K", [(8, 64, 4096), (64, 64, 8192), (200, 128, 16384), (2048, 64, 64), (4100, 72, 40)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_long_sums(M, N, K, dt):
    """Few outputs and a long reduction, forward (K) and in the weight's gradient (M)."""
    _check(*_inputs(M, N, K, dt, 3), "relu")


@pytest.mark.parametrize("M,N,K", [(700, 1200, 512), (1024, 1024, 1024), (520, 4096, 264)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_many_tiles(M, N, K, dt):
    _check(*_inputs(M, N, K, dt, 4), "gelu_tanh")


def _holed(t, pad):
    """t's values in rows `pad` elements longer, whose extra elements are NaN."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _shifted(t, by):
    """t's values `by` elements into an allocation whose other elements are NaN."""
    flat = torch.full((t.numel() + by + 3,), float("nan"), dtype=t.dtype, device=t.device)
    v = flat[by:by + t.numel()].view(t.shape)
    return v.copy_(t)


@pytest.mark.parametrize("M", [1, 7, 150])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("K", [64, 100, 72])
@pytest.mark.parametrize("pad", [1, 8])
def test_rows_with_holes(M, dt, K, pad):
    """Rows of x and weight that lie further apart; NaN between them stays out."""
    x, w, b, r, g = _inputs(M, 140, K, dt, 5)
    _check(_holed(x, pad), _holed(w, pad), b, r, g, "gelu")


@pytest.mark.parametrize("M", [1, 20, 150])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("by", [1, 2, 4])
def test_starts_off_a_vector(M, dt, by):
    x, w, b, r, g = _inputs(M, 136, 128, dt, 6)
    _check(_shifted(x, by), _shifted(w, by), _shifted(b, by), _shifted(r, by), _shifted(g, by), "silu")


@pytest.mark.parametrize("M", [6, 140])
def test_orders_and_leading_axes(M):
    x, w, b, r, g = _inputs(M, 72, 80, "bf16", 7)
    ref = linear_act(x, w, b, r, activation="gelu")
    assert torch.equal(linear_act(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t(), activation="gelu"), ref)
    y = linear_act(x.view(2, 1, M // 2, 80), w, b, r.view(2, 1, M // 2, 72), activation="gelu")
    assert y.shape == (2, 1, M // 2, 72) and torch.equal(y.view(M, 72), ref)
    one = linear_act(x[0], w, b, activation="gelu")
    assert one.shape == (72,) and torch.equal(one, linear_act(x[:1], w, b, activation="gelu")[0])
    # one row for every token: its gradient is the sum over them
    row = x[:1].clone().requires_grad_(True)
    out = linear_act(row.expand(M, 80), w, b, r, activation="gelu")
    out.backward(g)
    e, _, _, d, dz = linear64(row.expand(M, 80), w, b, r, "gelu", torch.bfloat16)
    (dx, bound), _, _ = linear_grads64(row.expand(M, 80), w, g, d, dz, torch.bfloat16, True)
    ones = torch.ones(1, M, dtype=torch.float64, device="cuda")
    s = ones @ dx
    # torch's sum over the tokens: rounded once more, from values that are each within their bound
    close(row.grad, s, ones @ bound + M * 2.0 ** -24 * (ones @ dx.abs()) + 2.0 ** -8 * s.abs(), "row")


def test_upstream_of_another_order_and_no_elements():
    x, w, b, r, g = _inputs(90, 72, 80, "bf16", 8)
    for t in (x, w, b, r):
        t.requires_grad_(True)
    a = torch.autograd.grad(linear_act(x, w, b, r, activation="silu"), (x, w, b, r), g)
    c = torch.autograd.grad(linear_act(x, w, b, r, activation="silu"), (x, w, b, r), g.t().contiguous().t())
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    one = torch.tensor(0.5, device="cuda", dtype=torch.bfloat16).expand(90, 72)
    a = torch.autograd.grad(linear_act(x, w, b, r, activation="silu"), (x, w), one)
    c = torch.autograd.grad(linear_act(x, w, b, r, activation="silu"), (x, w), one.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    e = torch.empty(3, 0, 80, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = linear_act(e, w, b, activation="silu")
    assert out.shape == (3, 0, 72)
    de, dw, db = torch.autograd.grad(out, (e, w, b), torch.empty_like(out))
    assert de.shape == e.shape and not dw.any() and not db.any()


def test_only_the_gradients_that_are_asked_for():
    x, w, b, r, g = _inputs(70, 72, 80, "f32", 9)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(linear_act(*full, activation="gelu"), full, g)
    for k in range(4):
        some = [t.clone().requires_grad_(j == k) for j, t in enumerate((x, w, b, r))]
        got, = torch.autograd.grad(linear_act(*some, activation="gelu"), some[k], g)
        assert torch.equal(got, want[k])


@pytest.mark.parametrize("act", ACTIVATIONS)
def test_against_differences(act):
    """Directional derivatives of sum(g out) in float64 differences of the plain form."""
    x, w, b, r, g = _inputs(9, 40, 24, "f32", 10)
    ts = [t.requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear_act(*ts, activation=act), ts, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for k, t in enumerate(ts):
        v = torch.randn(t.shape, generator=gen, device="cuda").double()
        h = 1e-6

        def value(e):
            args = [s.detach().double() + (e * v if j == k else 0.0) for j, s in enumerate(ts)]
            return (linear_act_reference(*args, activation=act) * g.double()).cpu().sum()

        slope = float(value(h) - value(-h)) / (2 * h)
        size = float((grads[k].double() * v).abs().cpu().sum())
        # differences: h^2 of a third derivative (relu: a kink passed within h |v|), 1e-16 / h of the value
        assert abs(float((grads[k].double() * v).cpu().sum()) - slope) <= 1e-5 * size + 1e-6


@pytest.mark.parametrize("M,N,K", [(4, 64, 96), (140, 136, 128), (140, 130, 100)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_non_finite_values_stay_in_their_rows(M, N, K, dt):
    x, w, b, r, _ = _inputs(M, N, K, dt, 11)
    clean = linear_act(x, w, b, r, activation="relu")
    x2 = x.clone()
    x2[1, K // 2] = float("nan")
    x2[3, 0] = float("inf")
    out = linear_act(x2, w, b, r, activation="relu")
    assert out[1].isnan().all() and not out[3].isfinite().all()
    keep = [i for i in range(M) if i not in (1, 3)]
    assert torch.equal(out[keep], clean[keep])
    w2 = w.clone()
    w2[N - 1, K - 1] = float("nan")
    out = linear_act(x, w2, b, r, activation="relu")
    assert out[:, N - 1].isnan().all() and torch.equal(out[:, :N - 1], clean[:, :N - 1])


@pytest.mark.parametrize("M,N,K", [(5, 64, 96), (100, 130, 96), (1024, 1600, 96), (2048, 2048, 104), (2100, 4300, 72)])
def test_fp32_extremes(M, N, K):
    """Infinities with their signs, and values near both ends of the range, in every row that has them and no other."""
    x, w, _, _, _ = _inputs(M, N, K, "f32", 17)
    x[1] *= 1e35
    x[2] *= 1e-34
    x[3, K - 1], x[4, 0] = float("inf"), -float("inf")
    w[5] *= 1e4
    w[6] *= 1e-4
    out = linear_act(x, w)
    ref, bound, *_ = linear64(x, w, None, None, "none", torch.float32)
    fine = ref.abs() < 3e38
    close(torch.where(fine, out.double(), 0.0), torch.where(fine, ref, 0.0), torch.where(fine, bound, 1.0), "finite")
    assert torch.equal(out[3:5].isinf(), ref[3:5].isinf()) and torch.equal(out[3:5].sign(), ref[3:5].sign().float())
    assert not out.isnan().any()


@pytest.mark.parametrize("M", [9, 70, 150, 700])
@pytest.mark.parametrize("dt,K", [("bf16", 4100), ("bf16", 4102), ("bf16", 4101), ("f32", 2049), ("f16", 1030)])
def test_ends_of_long_rows(M, dt, K):
    """Reductions that end inside a chunk, and inside a part where they are split; what follows each row in memory is NaN."""
    x, w, b, r, g = _inputs(M, 140, K, dt, 18)
    _check(_holed(x, 6), _holed(w, 10), b, r, g, "silu")


@pytest.mark.parametrize("N", [512, 516, 514, 513])
@pytest.mark.parametrize("dt,out", [("bf16", None), ("f16", torch.float32), ("f32", None)])
@pytest.mark.parametrize("M,K", [(300, 1000), (1030, 264), (2100, 200), (4200, 1032)])
def test_output_rows_of_any_length(M, N, K, dt, out):
    """Every tile, forward and backward, with outputs that end inside a vector."""
    N = N * 8 if M >= 2100 else N
    _check(*_inputs(M, N - (8 - N % 8) % 8 if N > 4000 else N, K, dt, 19, out=out), "gelu", out)


def test_more_than_2_31_elements():
    """Rows past 2^31 elements of x and past 2^32 bytes (a view of one allocation)."""
    M, K, N = 70000, 32768, 16
    x = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    x[:] = torch.randn(1, K, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    x[M - 200:] *= 2
    w = (torch.randn(N, K, device="cuda") * K ** -0.5).to(torch.bfloat16)
    out = linear_act(x, w)
    ref, bound, *_ = linear64(x[-300:], w, None, None, "none", torch.bfloat16)
    close(out[-300:], ref, bound, "last rows")
    assert torch.equal(out[:M - 200], out[:1].expand(M - 200, N))
    g = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    g[-100:] = 1.0
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_act(xg, wg), (xg, wg), g)
    assert not dx[:M - 100:997].any()
    (dx64, bx), (dw64, bw), _ = linear_grads64(x[-100:], w, g[-100:], torch.ones(100, N, device="cuda", dtype=torch.float64),
                                               torch.zeros(100, N, device="cuda", dtype=torch.float64), torch.bfloat16, False)
    close(dx[-100:], dx64, bx, "dx")
    close(dw, dw64, bw + M * 2.0 ** -24 * (torch.ones(N, 100, device="cuda", dtype=torch.float64) @ x[-100:].double().abs()), "dw")


def test_on_another_stream_and_in_a_graph():
    x, w, b, r, g = _inputs(150, 264, 192, "bf16", 12)
    ts = [t.requires_grad_(True) for t in (x, w, b, r)]

    def step():
        out = linear_act(*ts, activation="gelu")
        return (out.detach(), *torch.autograd.grad(out, ts, g))

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
            x.add_(0.25)
            for t in held[:-1]:  # (the last is the residual's gradient: g itself)
                t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step())), k


def test_results_repeat():
    x, w, b, r, g = _inputs(333, 520, 4096, "bf16", 13)
    ts = [t.requires_grad_(True) for t in (x, w, b, r)]
    runs = []
    for _ in range(3):
        out = linear_act(*ts, activation="gelu")
        runs.append((out.detach(), *torch.autograd.grad(out, ts, g)))
    assert all(torch.equal(p, q) for run in runs[1:] for p, q in zip(run, runs[0]))


def test_timer_and_trace_take_the_same_kernels():
    x, w, b, r, g = _inputs(20, 64, 48, "bf16", 14)
    ts = [t.requires_grad_(True) for t in (x, w, b, r)]
    out = linear_act(*ts, activation="silu")
    want = torch.autograd.grad(out, ts, g)
    with kernel_timer() as kt:
        timed = linear_act(*ts, activation="silu")
        got = torch.autograd.grad(timed, ts, g)
    assert set(kt.stats()) == {"linear_act_fwd", "linear_act_bwd"}
    assert torch.equal(timed, out) and all(torch.equal(p, q) for p, q in zip(got, want))
    m = FusedLinear(48, 64, activation="silu", device="cuda", dtype=torch.bfloat16)
    traced = torch.jit.trace(m, (x.detach(),), check_trace=False)
    other = torch.randn(20, 48, device="cuda").to(torch.bfloat16)
    for t in (x.detach(), other):
        assert torch.equal(traced(t), m(t))


def test_second_derivatives_are_refused():
    x, w, b, _, g = _inputs(5, 16, 8, "f32", 15)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(linear_act(x, w, b, activation="gelu"), x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.square().sum().backward()


def test_refusals():
    x, w, b, r, _ = _inputs(5, 16, 8, "bf16", 16)
    for bad in [dict(x=x.cpu()), dict(weight=w.cpu()), dict(x=x.float()), dict(bias=b.float()), dict(bias=b[:-1]), dict(bias=b[None]),
                dict(residual=r[:-1]), dict(residual=r.float()), dict(weight=w[:, :-1]), dict(weight=w[0]), dict(activation="tanh"),
                dict(activation=None), dict(output_dtype=torch.float16), dict(x=x.double(), weight=w.double()),
                dict(x=x[:, :0], weight=w[:, :0]), dict(weight=w[:0]), dict(output_dtype=torch.float64),
                dict(residual=r, output_dtype=torch.float32)]:
        args = dict(x=x, weight=w, bias=None, residual=None, activation="none", output_dtype=None) | bad
        with pytest.raises(ValueError):
            linear_act(**args)


@pytest.mark.parametrize("n", [4, 16])
def test_fused_linear_inside_mhc_rewire(n):
    """MHCRewire around FusedLinear against the same wrapper around a float32 Linear of the same weights."""
    lin = FusedLinear(128, 128, device="cuda")
    plain = torch.nn.Linear(128, 128, device="cuda")
    plain.load_state_dict(lin.state_dict())
    a, b = (MHCRewire(m, 128, n, identity_init=False).cuda() for m in (lin, plain))
    x = torch.randn(300, 128, device="cuda")
    ya, yb = a(x), b(x)
    # one product of 128 terms each
    assert (ya - yb).abs().max() <= 4 * 130 * 2.0 ** -24 * yb.abs().max()
    model = torch.nn.Sequential(FusedLinear(64, 64, activation="relu"), torch.nn.Linear(64, 64)).cuda()
    assert AutoPatcher.patch(model, n_streams=4, verbose=False) == 2
    model(torch.randn(3, 64, device="cuda")).sum().backward()
    assert model[0].inner.weight.grad is not None


def test_module_forms():
    m = FusedLinear(24, 40, activation="gelu", return_dtype=torch.float32, device="cuda", dtype=torch.bfloat16)
    x, r = torch.randn(7, 24, device="cuda").to(torch.bfloat16), torch.randn(7, 40, device="cuda")
    out = m(x, r)
    ref, bound, *_ = linear64(x, m.weight, m.bias, r, "gelu", torch.float32)
    assert out.dtype == torch.float32
    close(out, ref, bound)
    y, d = act64(ref, "none")
    assert y.shape == d.shape


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [17, 32, 64])
@pytest.mark.parametrize("columns,more", [(16, 0), (16, 2), (25, 7), (32, 0), (32, 1)])
def test_few_rows_of_wide_layers(M, columns, more, dt):
    """Around the widths that give each compute unit one workgroup of 16 or of 32 columns."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    _check(*_inputs(M, columns * cus + more, 200, dt, 21), "gelu")


@pytest.mark.parametrize("M,N,K", [(70, 300, 200), (100, 2048, 72), (90, 72, 2048), (512, 512, 1024), (1000, 520, 1030), (1500, 1001, 260),
                                   (2049, 1500, 1024), (3000, 200, 130)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bias", [True, False])
def test_backward_of_middle_sizes(M, N, K, dt, bias):
    """Both products of the backward in one launch, whole and split, with and without the bias's sums."""
    ts = _inputs(M, N, K, dt, 22, bias=bias)
    _check(*ts, "silu")
    x, w, b, _, g = ts

    def grads():
        return torch.autograd.grad(linear_act(x, w, b, activation="silu"), [t for t in (x, w, b) if t is not None], g)

    for one, two in zip(grads(), grads()):
        assert torch.equal(one, two)
