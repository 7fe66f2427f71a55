"""linear_cross_entropy on the GPU against float64 (tests/_block.py)."""

import ctypes

import pytest
import torch

from mhc_mlx_amd import AddRMSNorm, FusedLinear, _lib, kernel_timer, linear_cross_entropy, linear_cross_entropy_and_grad, ops, policy_loss
from tests._block import ce64
from tests._train import close

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def inputs(seed, T, V, C, dt, near=3.0):
    g = gen(seed)
    w = (torch.randn(V, C, generator=g, device="cuda") * C ** -0.5).to(dt)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    x = (torch.randn(T, C, generator=g, device="cuda") + near * w[y].float()).to(dt)
    return x, w, y, g


def check(x, w, y, mask=None, den=None, scale=1.0, what="", **kw):
    ref = ce64(x, w, y, mask, den, scale=scale, **kw)
    got = dict(zip(("loss", "logp", "dx", "dw"), linear_cross_entropy_and_grad(x, w, y, mask, den, grad_scale=scale, **kw)))
    assert got["dx"].dtype == got["dw"].dtype == x.dtype
    for k, (value, bound) in ref.items():
        close(got[k], value, bound, f"{what} {k}")
    xs, ws = (t.detach().requires_grad_(True) for t in (x, w))
    loss, logp = linear_cross_entropy(xs, ws, y, mask, den, **kw)
    assert torch.equal(loss, got["loss"]) and torch.equal(logp, got["logp"])
    dx, dw = torch.autograd.grad(loss, [xs, ws], torch.tensor(scale, device="cuda"))
    close(dx, *ref["dx"], f"{what} dx")
    close(dw, *ref["dw"], f"{what} dw")
    return got


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,V,C", [(1, 1, 1), (1, 2, 8), (2, 65, 7), (5, 64, 16), (17, 1000, 33), (64, 257, 64), (65, 129, 100), (130, 515, 72),
                                   (300, 2050, 128), (700, 1003, 250), (33, 5000, 515)])
def test_loss_and_gradients(dt, T, V, C):
    x, w, y, g = inputs(T + V, T, V, C, dt)
    check(x, w, y, what="all")
    mask = torch.rand(T, generator=g, device="cuda") < 0.6
    check(x, w, y, mask, scale=256.0, what="mask")
    check(x, w, y, torch.randn(T, generator=g, device="cuda") * mask, den=3.0, what="weights")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,V,C", [(1024, 4096, 256), (2050, 3001, 512), (520, 20000, 64), (3000, 500, 1000)])
def test_larger_tiles_and_splits(dt, T, V, C):
    x, w, y, g = inputs(T, T, V, C, dt)
    check(x, w, y, torch.rand(T, generator=g, device="cuda") < 0.75)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_vocabularies_of_several_pieces(dt):
    """dz of 5000 tokens over 30011 columns is more than a piece: dx is summed up over them, dw written piece by piece."""
    x, w, y, g = inputs(3, 5000, 30011, 40, dt)
    y[:7] = torch.tensor([0, 30010, 255, 256, 15103, 15104, 30000], device="cuda")
    check(x, w, y, torch.rand(5000, generator=g, device="cuda") < 0.9)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 5, 8, 9, 16])
def test_few_tokens(dt, T):
    """dx and dW in one pass over W: widths off every vector's length, rows that start anywhere, one column of the vocabulary."""
    for V, C in ((1000, 2285), (5003, 300), (40, 4100), (1, 33), (33, 1), (70001, 24)):
        x, w, y, g = inputs(T + C, T, V, C, dt)
        mask = torch.rand(T, generator=g, device="cuda") < 0.7
        check(x, w, y, scale=64.0, what=f"{V} {C}")
        got = check(x, w, y, mask, what=f"{V} {C} mask")
        # what lies between rows and behind them is not looked at
        wide = torch.full((V + 1, C + 5), float("nan"), device="cuda", dtype=dt)
        wv, xv = wide[:V, 3:C + 3].copy_(w), torch.full((T, C + 7), float("nan"), device="cuda", dtype=dt)[:, 1:C + 1].copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(xv, wv, y, mask), got.values()))
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(linear_cross_entropy(xs, w, y, mask)[0], xs)[0], got["dx"])
        assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, ws, y, mask)[0], ws)[0], got["dw"])
        none = check(x, w, y, torch.zeros(T, device="cuda"), what="no token")
        assert not none["dx"].any() and not none["dw"].any()
    y2 = y.clone()
    y2[0] = V
    loss, logp, dx, dw = linear_cross_entropy_and_grad(x, w, y2)
    assert bool(loss.isnan()) and bool(dx[0].isnan().all()) and bool(dx[1:].isfinite().all()) and bool(dw.isnan().all())


def at_the_c_abi(x, w, y, mask, keep, scale=1.0):
    """The two calls with the logits kept between them or formed again, whatever the sizes."""
    lib, byref, T, V = _lib.load(), ctypes.byref, len(x), len(w)
    pitch = -(-V // 64) * 64
    logits = torch.full((T * pitch + 64,), float("nan"), device="cuda") if keep else None
    a = _lib.LinearCeArgs(x=x.data_ptr(), ldx=x.stride(0), w=w.data_ptr(), ldw=w.stride(0), targets=y.data_ptr(), weights=mask.data_ptr(), weights_dtype=3, T=T, V=V,
                          C=x.shape[1], dtype=ops._code(x.dtype), ignore_index=-100, denominator=0.0, logits=logits.data_ptr() if keep else None)
    new = lambda n: torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")  # noqa: E731
    s, loss, logp = torch.cuda.current_stream().cuda_stream, torch.empty((), device="cuda"), torch.empty(T, device="cuda")
    state = new(lib.mhc_linear_ce_state_bytes(T))
    nf, nb = lib.mhc_linear_ce_fwd_workspace_bytes(byref(a)), lib.mhc_linear_ce_bwd_workspace_bytes(byref(a), 1, 1)
    assert lib.mhc_linear_ce_logits_bytes(byref(a)) in (0, T * pitch * 4)
    assert lib.mhc_linear_ce_fwd(byref(a), loss.data_ptr(), logp.data_ptr(), state.data_ptr(), new(nf).data_ptr(), nf, s) == 0
    outs = []
    for _ in range(2):  # (the backward leaves the logits as they are)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        assert lib.mhc_linear_ce_bwd(byref(a), state.data_ptr(), None, ctypes.c_float(scale), dx.data_ptr(), dw.data_ptr(), new(nb).data_ptr(), nb, s) == 0
        outs.append((dx, dw))
    assert all(torch.equal(p, q) for p, q in zip(*outs))
    assert not keep or bool(logits[T * pitch:].isnan().all())
    return dict(loss=loss, logp=logp, dx=dx, dw=dw)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,V,C", [(1, 2, 8), (2, 65, 8), (17, 1000, 40), (64, 257, 64), (130, 515, 72), (300, 2050, 128), (700, 1003, 256), (1024, 4096, 256),
                                   (2050, 3001, 512), (520, 20000, 64), (3000, 500, 1000), (5000, 30011, 40), (4500, 30011, 256), (700, 5003, 1030), (2500, 30011, 520), (300, 9000, 2051)])
def test_logits_kept_and_formed_again(dt, T, V, C):
    x, w, y, g = inputs(T + V, T, V, C, dt)
    mask = (torch.rand(T, generator=g, device="cuda") < 0.8).to(torch.uint8)
    ref = ce64(x, w, y, mask, scale=16.0)
    for keep in (True, False):
        for k, v in at_the_c_abi(x, w, y, mask, keep, 16.0).items():
            close(v, *ref[k], f"{k} kept {keep}")


def test_gradients_of_huge_weights_over_several_pieces():
    """Weights around 2^112, whose sums in dx are formed a second time, are added to those of the pieces before."""
    x, w, y, _ = inputs(16, 5000, 30011, 256, torch.float32)
    x, w = x * 2.0 ** -112, w * 2.0 ** 112
    check(x, w, y)
    ref = ce64(x, w, y)
    for k, v in at_the_c_abi(x, w, y, torch.ones(5000, dtype=torch.uint8, device="cuda"), False).items():
        close(v, *ref[k], f"{k} of logits formed again")


@pytest.mark.parametrize("dt", DTYPES)
def test_tokens_left_out(dt):
    x, w, y, g = inputs(5, 200, 333, 48, dt)
    full = check(x, w, y)
    # nothing of a token that is left out counts, whatever it holds
    mask = torch.rand(200, generator=g, device="cuda") < 0.5
    clean = check(x, w, y, mask)
    x2, y2 = x.clone(), y.clone()
    x2[~mask] = float("nan")
    y2[~mask] = 10 ** 12
    dirty = linear_cross_entropy_and_grad(x2, w, y2, mask)
    assert all(torch.equal(a, b) for a, b in zip(dirty, clean.values()))
    assert not clean["dx"][~mask].any() and not clean["logp"][~mask].any()
    # an ignored target is as good as a mask
    y3 = torch.where(mask, y, -100)
    assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(x2, w, y3), clean.values()))
    assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(x2, w, torch.where(mask, y, 7), mask, ignore_index=-5), linear_cross_entropy_and_grad(x, w, y, mask)))
    # bytes and floats as masks, int32 targets
    for m in (mask.to(torch.uint8) * 3, mask.half(), mask.double()):
        assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(x, w, y.int(), m), clean.values()))
    # no token at all, and one
    for m in (torch.zeros(200, device="cuda"), torch.arange(200, device="cuda") == 150):
        got = check(x, w, y, m)
        assert bool(got["dw"].isfinite().all())
    assert float(linear_cross_entropy(x, w, y, torch.zeros(200, device="cuda"))[0]) == 0.0
    assert full["loss"] > 0


@pytest.mark.parametrize("dt", DTYPES)
def test_targets_out_of_range_and_nan(dt):
    x, w, y, _ = inputs(6, 70, 100, 32, dt)
    for bad in (-1, 100, 2 ** 40, -2 ** 62):
        y2 = y.clone()
        y2[3] = bad
        loss, logp, dx, dw = linear_cross_entropy_and_grad(x, w, y2)
        others = torch.arange(70, device="cuda") != 3
        assert bool(loss.isnan()) and bool(logp[3].isnan()) and bool(logp[others].isfinite().all())
        assert bool(dx[3].isnan().all()) and bool(dx[others].isfinite().all()) and bool(dw.isnan().all())
    x2 = x.clone()
    x2[5, 2] = float("nan")
    loss, logp, dx, _ = linear_cross_entropy_and_grad(x2, w, y)
    others = torch.arange(70, device="cuda") != 5
    assert bool(loss.isnan()) and bool(dx[5].isnan().all()) and bool(dx[others].isfinite().all()) and bool(logp[others].isfinite().all())


@pytest.mark.parametrize("dt", DTYPES)
def test_logits_far_apart(dt):
    """Logits of up to some 10^4 with one that takes all, and rows whose logits are all alike."""
    x, w, y, _ = inputs(7, 60, 500, 64, dt)
    check((x * 2000).to(dt), w, y, what="large")
    check(torch.zeros_like(x), w, y, what="alike")


@pytest.mark.parametrize("T,V,C", [(40, 300, 64), (1024, 4096, 256), (1500, 4096, 1100)])
def test_fp32_rows_of_many_magnitudes(T, V, C):
    """Few tokens and many (whose logits are products of fp16 parts): rows from 2^-60 to 2^8 times the usual, one of zeros, one subnormal."""
    x, w, y, g = inputs(15, T, V, C, torch.float32)
    x = x * 2.0 ** torch.randint(-60, 9, (T, 1), generator=g, device="cuda").float()
    w = w * 2.0 ** torch.randint(-40, 3, (V, 1), generator=g, device="cuda").float()
    x = x * 2.0 ** torch.randint(-10, 1, (1, C), generator=g, device="cuda").float()  # (and values of a row)
    x[3], w[7] = 0.0, 0.0
    x[4], w[8] = x[4] * 2.0 ** -100, w[8] * 2.0 ** -90
    check(x, w, y, what="magnitudes")
    x[5, 1] = float("inf")
    loss, logp, dx, _ = linear_cross_entropy_and_grad(x, w, y)
    others = torch.arange(T, device="cuda") != 5
    assert bool(loss.isnan()) and bool(logp[5].isnan()) and bool(logp[others].isfinite().all()) and bool(dx[others].isfinite().all())


@pytest.mark.parametrize("T,V,C,by", [(40, 300, 64, 105), (1024, 4096, 256, 118), (1500, 4096, 1100, 118)])
def test_fp32_operands_that_are_large_and_small(T, V, C, by):
    """Logits of the usual size from rows around 2^by and weights around 2^-by, and the other way round."""
    x, w, y, _ = inputs(18, T, V, C, torch.float32)
    for up in (by, -by):
        check(x * 2.0 ** up, w * 2.0 ** -up, y, what=f"{up}")


def test_strides_and_shapes():
    x, w, y, g = inputs(8, 60, 90, 64, torch.bfloat16)
    want = linear_cross_entropy_and_grad(x, w, y)
    wide = torch.zeros(60, 100, device="cuda", dtype=torch.bfloat16)
    for at in (0, 3, 8):
        xv = wide[:, at:at + 64].copy_(x)
        wv = torch.zeros(90, 101, device="cuda", dtype=torch.bfloat16)[:, at:at + 64].copy_(w)
        assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(xv, wv, y), want))
    wt = w.t().contiguous().t()
    shaped = linear_cross_entropy_and_grad(x.view(3, 4, 5, 64), wt, y.view(3, 4, 5))
    assert shaped[1].shape == (3, 4, 5) and shaped[2].shape == (3, 4, 5, 64) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(shaped, want))
    one = linear_cross_entropy(x[0], w, y[0])
    assert one[1].shape == () and torch.equal(one[1], want[1][0])
    e = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ww = w.clone().requires_grad_(True)
    loss, logp = linear_cross_entropy(e, ww, y[:0])
    loss.backward()
    assert float(loss) == 0 and logp.shape == (0,) and not ww.grad.any() and e.grad.shape == (0, 64)


def test_which_gradients_are_asked_for():
    x, w, y, _ = inputs(9, 90, 300, 72, torch.float32)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, logp = linear_cross_entropy(xs, ws, y)
    assert not logp.requires_grad
    dx, dw = torch.autograd.grad(loss, [xs, ws])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(xs, w, y)[0], xs)[0], dx)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(x, ws, y)[0], ws)[0], dw)
    with kernel_timer() as kt:
        timed = torch.autograd.grad(linear_cross_entropy(xs, ws, y)[0], [xs, ws])
    assert torch.equal(timed[0], dx) and torch.equal(timed[1], dw) and "linear_cross_entropy_bwd" in kt.stats()
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        d, = torch.autograd.grad(linear_cross_entropy(xs, ws, y)[0], xs, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("dt", DTYPES)
def test_against_kept_logits(dt):
    """FusedLinear's logits and policy_loss with a ratio of one: its log probabilities are these."""
    x, w, y, _ = inputs(10, 100, 1000, 256, dt)
    head = FusedLinear(256, 1000, bias=False, device="cuda", dtype=dt, return_dtype=torch.float32)
    with torch.no_grad():
        head.weight.copy_(w)
        logp = policy_loss(head(x), y, torch.zeros(100, device="cuda"), torch.ones(100, device="cuda"))[1]
    ours = linear_cross_entropy(x, w, y)[1]
    assert float((logp - ours).abs().max()) < 2e-5 * float(logp.abs().max())


def test_a_head_with_its_norm_learns_as_the_formula_says():
    """add_rms_norm into the loss, both with their gradients, against float64."""
    g = gen(11)
    T, V, C = 300, 700, 128
    norm = AddRMSNorm(C, device="cuda")
    x, r = (torch.randn(T, C, generator=g, device="cuda").requires_grad_(True) for _ in range(2))
    w = (torch.randn(V, C, generator=g, device="cuda") * 0.1).requires_grad_(True)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    n, h = norm(x, r)
    loss, _ = linear_cross_entropy(n, w, y)
    (loss + (h * h).mean()).backward()
    xd, rd, wd, gd = (t.detach().double().requires_grad_(True) for t in (x, r, w, norm.weight))
    hd = xd + rd
    nd = hd / torch.sqrt((hd * hd).mean(1, keepdim=True) + norm.eps) * gd
    z = nd @ wd.t()
    ref = (torch.logsumexp(z, 1) - z.gather(1, y[:, None])[:, 0]).mean()
    (ref + (hd * hd).mean()).backward()
    assert abs(float(loss) - float(ref)) < 1e-5
    for a, b in ((x, xd), (r, rd), (w, wd), (norm.weight, gd)):
        assert float((a.grad - b.grad).norm() / b.grad.norm()) < 1e-5


def test_refusals():
    x, w, y, _ = inputs(12, 10, 20, 16, torch.bfloat16)
    for args in ((x.float(), w, y), (x, w[:, :8], y), (x, w, y[:9]), (x, w, y.float()), (x.cpu(), w, y), (x, w.cpu(), y), (x, w, y.cpu()), (x.double(), w.double(), y),
                 (x, w[0], y), (x, w[:0], y), (x, w, y, torch.ones(9, device="cuda")), (x, w, y, torch.ones(10, device="cuda", dtype=torch.int32)),
                 (x, w, y, None, 0.0), (x, w, y, None, -1.0)):
        with pytest.raises(ValueError):
            linear_cross_entropy(*args)
        with pytest.raises(ValueError):
            linear_cross_entropy_and_grad(*args)


def test_the_same_call_twice_and_on_another_stream():
    x, w, y, g = inputs(13, 2000, 5000, 256, torch.bfloat16)
    mask = torch.rand(2000, generator=g, device="cuda") < 0.7
    a = linear_cross_entropy_and_grad(x, w, y, mask)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = linear_cross_entropy_and_grad(x, w, y, mask)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", DTYPES)
def test_a_backward_twice(dt):
    """Logits that are kept stay as they are until the graph is freed; without a gradient the loss is the same."""
    x, w, y, _ = inputs(17, 130, 700, 776, dt)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss, logp = linear_cross_entropy(xs, ws, y)
    a = torch.autograd.grad(loss, [xs, ws], retain_graph=True)
    b = torch.autograd.grad(loss, [xs, ws])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    plain = linear_cross_entropy(x, w, y)
    assert torch.equal(plain[0], loss) and torch.equal(plain[1], logp)


@pytest.mark.parametrize("C", [128, 800])
def test_captured_calls_with_other_masks(C):
    """How many tokens count is found on the device: a graph's replays follow the mask."""
    x, w, y, g = inputs(14, 300, 1000, C, torch.bfloat16)
    mask = torch.ones(300, device="cuda")

    def step():
        xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss, logp = linear_cross_entropy(xs, ws, y, mask)
        return [loss.detach(), logp, *torch.autograd.grad(loss, [xs, ws])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for share in (0.5, 0.0, 1.0, 0.1):
        mask.copy_(torch.rand(300, generator=g, device="cuda") < share)
        x.normal_(generator=g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), share


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,C", [(6, 1000, 300), (16, 3001, 129), (900, 4000, 1024)])
def test_captured_calls_of_few_tokens_and_of_parts(dt, T, V, C):
    x, w, y, g = inputs(19, T, V, C, dt)
    mask = torch.ones(T, device="cuda")

    def step():
        xs, ws = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss, logp = linear_cross_entropy(xs, ws, y, mask)
        return [loss.detach(), logp, *torch.autograd.grad(loss, [xs, ws])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for share in (0.5, 0.0, 1.0):
        mask.copy_(torch.rand(T, generator=g, device="cuda") < share)
        x.normal_(generator=g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), share


def test_calls_from_two_threads():
    """Each on a stream of its own, with operands of its own."""
    import threading

    cases = [inputs(20, 5, 3000, 512, torch.float32)[:3], inputs(21, 900, 2000, 1024, torch.float32)[:3], inputs(22, 700, 3000, 800, torch.bfloat16)[:3]]
    want = [linear_cross_entropy_and_grad(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                for k in order:
                    got = linear_cross_entropy_and_grad(*cases[k])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append(k)

    threads = [threading.Thread(target=work, args=(o,)) for o in ((0, 1, 2), (2, 1, 0))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
