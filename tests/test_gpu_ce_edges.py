"""linear_cross_entropy at the ends of fp32's range, where its products are of fp16 parts: against float64 (tests/_block.py)."""

import pytest
import torch

from mhc_mlx_amd import kernel_timer, linear_cross_entropy, linear_cross_entropy_and_grad
from tests._block import ce64
from tests._train import close

pytestmark = pytest.mark.gpu

# fp32 sizes whose logits are kept and whose gradients are formed of parts
PARTS = [(900, 4000, 1024), (1100, 32768, 1024)]


def rand(seed, *shapes):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=g, device="cuda") for s in shapes]


def check(x, w, y, what, scale=1.0):
    """Against ce64, and what parts cannot hold: terms are lifted by at most 2^126 to fp16 parts, whose least step is 2^-24, and meet
    parts of up to 2^15, so that each of a sum's products is off by half of 2^-24 2^-126 2^15 at most, for each of two operands."""
    got = dict(zip(("loss", "logp", "dx", "dw"), linear_cross_entropy_and_grad(x, w, y, grad_scale=scale)))
    least = scale / len(y) * 2.0 ** -135
    for k, (value, bound) in ce64(x, w, y, scale=scale).items():
        close(got[k], value, bound + {"dx": len(w), "dw": len(y)}.get(k, 0) * least, f"{what} {k}")


@pytest.mark.parametrize("T,V,C", PARTS)
@pytest.mark.parametrize("up", [15, 16, 20, 40])
def test_columns_without_probability(T, V, C, up):
    """Rows of x around 2^up: nearly every column's probabilities are 0, and its gradient with them."""
    x, w = rand(up, (T, C), (V, C))
    y = torch.arange(T, device="cuda") % V
    check(x * 2.0 ** (up - 1), w * C ** -0.5, y, f"x {up}")


@pytest.mark.parametrize("T,V,C", PARTS)
@pytest.mark.parametrize("up", [16, 20, 40])
def test_tokens_that_are_certain(T, V, C, up):
    """Rows of W around 2^up, some tokens near their targets' rows: their probability is 1, their dz 0 everywhere."""
    x, w = rand(up, (T, C), (V, C))
    y = torch.arange(T, device="cuda") * 3 % V
    w = w * 2.0 ** (up - 1)
    x[::2] += 4.0 * 2.0 ** (1 - up) * w[y[::2]]
    check(x, w, y, f"w {up}")


@pytest.mark.parametrize("up", [0, 16, 40, 100, -100])
def test_probabilities_that_are_subnormal(up):
    """All tokens' probabilities of each column but one between e^-83 and e^-105, beside rows of x or of W around 2^|up|."""
    T, V, C = 900, 4000, 1024
    noise, = rand(7, (T, C))
    along = torch.ones(C, device="cuda") / C ** 0.5
    below = -(85.0 + 18.0 * torch.arange(V, device="cuda") / V)
    below[0] = 0.0
    x = (along + 0.001 * noise) * 2.0 ** up
    w = (below[:, None] * along) * 2.0 ** -up
    y = torch.zeros(T, dtype=torch.int64, device="cuda")
    scale = 1.0 if abs(up) == 100 else 2.0 ** 40  # (so that gradients are neither past the range nor subnormal)
    check(x, w, y, f"{up}", scale)
    y[::3] = 1 + torch.arange(T, device="cuda")[::3]
    check(x, w, y, f"{up} with unlikely targets", scale)


@pytest.mark.parametrize("T,V,C", PARTS + [(700, 32768, 128)])
def test_large_rows_that_meet_in_no_element(T, V, C):
    """Rows of x around 2^100 and of W around 2^80 whose products are 0, beside ordinary ones: logits are those of the formula.  (dx and
    dW hold their terms to 2^-40 of the largest ones, which the large rows' are.)"""
    x, w = rand(3, (T, C), (V, C))
    w *= C ** -0.5
    x[:, :2], w[:, :2] = 0.0, 0.0
    x[5], w[7] = 0.0, 0.0
    x[5, 0], w[7, 1] = 2.0 ** 100, -2.0 ** 80
    y = torch.arange(T, device="cuda")
    loss, logp, dx, dw = linear_cross_entropy_and_grad(x, w, y)
    ref = ce64(x, w, y)
    close(loss, *ref["loss"], "loss")
    close(logp, *ref["logp"], "logp")
    assert bool(dx.isfinite().all()) and bool(dw.isfinite().all())


@pytest.mark.parametrize("given", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_under_autocast(dt, given):
    """Operands of two dtypes are taken in the autocast one; gradients come in their own."""
    x, w = rand(9, (70, 96), (300, 96))
    x, w = x.to(given[0]).requires_grad_(True), (w * 0.1).to(given[1]).requires_grad_(True)
    y = torch.arange(70, device="cuda")
    cast = dt if given[0] != given[1] else given[0]
    xs, ws = x.detach().to(cast).requires_grad_(True), w.detach().to(cast).requires_grad_(True)
    want = linear_cross_entropy(xs, ws, y)
    dx, dw = torch.autograd.grad(want[0], [xs, ws])
    with torch.autocast("cuda", dt):
        got = linear_cross_entropy(x, w, y)
        fused = linear_cross_entropy_and_grad(x, w, y)
    grads = torch.autograd.grad(got[0], [x, w])
    assert grads[0].dtype == x.dtype and grads[1].dtype == w.dtype
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(grads[0], dx.to(x.dtype)) and torch.equal(grads[1], dw.to(w.dtype))
    assert all(torch.equal(a, b) for a, b in zip(fused, (want[0], want[1], *grads)))
    if cast != given[0] or cast != given[1]:
        with pytest.raises(ValueError, match="dtype"):
            linear_cross_entropy(x, w, y)


def test_other_operands_under_autocast_are_refused():
    x, w = rand(10, (4, 16), (8, 16))
    y = torch.arange(4, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        for a, b in ((x, w.double()), (x.double(), w), (x, w.int()), (x.bfloat16(), w.to(torch.float8_e4m3fn).view(torch.uint8))):
            with pytest.raises(ValueError):
                linear_cross_entropy(a, b, y)
            with pytest.raises(ValueError):
                linear_cross_entropy_and_grad(a, b, y)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 3, 8, 9, 16])
def test_few_tokens_over_a_vocabulary_that_tiles_read_faster(T, dt):
    """Strides, tokens left out, none at all, and a captured call that follows its mask."""
    V, C = 32000, 2048
    x, w = rand(T, (T, C), (V, C))
    w = (w * C ** -0.5).to(dt)
    y = (torch.arange(T, device="cuda") * 1999 + 7) % V
    x = (x + 3.0 * w[y].float()).to(dt)
    mask = torch.arange(T, device="cuda") % 3 != 1
    want = linear_cross_entropy_and_grad(x, w, y, mask, grad_scale=64.0)
    for got, (value, bound) in zip(want, ce64(x, w, y, mask, scale=64.0).values()):
        close(got, value, bound)
    wide = torch.full((T, C + 9), float("nan"), device="cuda", dtype=dt)
    for at in (0, 1, 4):
        xv = wide[:, at:at + C].copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(xv, w, y, mask, grad_scale=64.0), want))
    xm = torch.where(mask[:, None], x, float("nan"))
    assert all(torch.equal(a, b) for a, b in zip(linear_cross_entropy_and_grad(xm, w, y, mask, grad_scale=64.0), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        linear_cross_entropy(x, w, y, mask)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = linear_cross_entropy(x, w, y, mask)
    for m in (mask, ~mask, torch.zeros_like(mask), torch.ones_like(mask)):
        mask.copy_(m.clone())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, linear_cross_entropy(x, w, y, mask)))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [6, 700])
def test_logits_that_are_not_to_be_kept(dt, T):
    """What lies between forward and backward does not grow with the vocabulary; gradients are within the same bounds."""
    V, C = 20000, 1024
    x, w = rand(T, (T, C), (V, C))
    w = (w * C ** -0.5).to(dt)
    y = torch.arange(T, device="cuda") * 17 % V
    x = (x + 3.0 * w[y].float()).to(dt)
    ref = ce64(x, w, y)
    xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    held = {}
    for keep in (True, False):
        before = torch.cuda.memory_allocated()
        loss, logp = linear_cross_entropy(xs, ws, y, keep_logits=keep)
        held[keep] = torch.cuda.memory_allocated() - before
        dx, dw = torch.autograd.grad(loss, [xs, ws])
        fused = linear_cross_entropy_and_grad(x, w, y, keep_logits=keep)
        with kernel_timer():
            timed = linear_cross_entropy(xs, ws, y, keep_logits=keep)
            grads = torch.autograd.grad(timed[0], [xs, ws])
        for k, (value, bound) in ref.items():
            close(dict(loss=loss, logp=logp, dx=dx, dw=dw)[k], value, bound, f"{k} {keep}")
        assert all(torch.equal(a, b) for a, b in zip(fused, (loss, logp, dx, dw)))
        assert all(torch.equal(a, b) for a, b in zip((*timed, *grads), (loss, logp, dx, dw)))
    assert held[True] >= T * V * 4 and held[False] < 64 * T + 4096
