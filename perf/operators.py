"""The operators of a training step around the mHC layer, on one GPU: what is measured of them, and their plain forms.

Three kinds of case, one for each operator:

  linear   linear_act: a matrix product with bias, activation and residual; a call without gradients, or a training step's call and backward
  policy   policy_loss / policy_loss_and_grad: the clipped policy loss with a KL term, from the logits
  adamw    adamw_step_hip: one AdamW step over a list of tensors, states in 32 or in 8 bits

With ``own`` false, ``run`` computes them from elementary torch operations in fp32; with ``own`` true, through mhc_mlx_amd.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
BETAS, EPS, LR, DECAY, STEP = (0.9, 0.95), 1e-8, 3e-4, 0.1, 100
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
BLOCK = 256  # elements of an 8-bit state that share a scale; every tensor starts at a multiple of it in the flat buffers


def _linear(M, N, K, dtype, act, train=False, bias=True, residual=True):
    return {"kind": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "act": act, "train": train, "bias": bias, "residual": residual}


def _policy(T, V, dtype, form, masked=0.25, pad=0, kl=0.05, scale=1.0):
    return {"kind": "policy", "T": T, "V": V, "dtype": dtype, "form": form, "masked": masked, "pad": pad, "kl": kl, "scale": scale}


def _adamw(layers, n, C, rows, cols, dtype, master=False, bits=32):
    return {"kind": "adamw", "layers": layers, "n": n, "C": C, "rows": rows, "cols": cols, "dtype": dtype, "master": master, "bits": bits}


def listed():
    return [
        # one token through a square layer of a block: bound by reading the weight, latency counts
        dict(_linear(1, 4096, 4096, "bf16", "gelu"), name="linear_1x4096x4096_bf16"),
        # a decoding step of a small batch through the widening product of a feed-forward block
        dict(_linear(32, 8192, 2048, "fp16", "silu", residual=False), name="linear_32x8192x2048_fp16"),
        # a prompt of odd length at a width that is no multiple of a vector
        dict(_linear(1001, 2050, 1100, "bf16", "relu"), name="linear_1001x2050x1100_bf16"),
        # prefill of a large batch through the widening product
        dict(_linear(16384, 16384, 4096, "bf16", "gelu_tanh", residual=False), name="linear_16384x16384x4096_bf16"),
        # a training step's call of the layer that MHCRewire wraps: 8192 tokens, forward and every gradient
        dict(_linear(8192, 4096, 4096, "bf16", "gelu", train=True), name="linear_train_8192x4096x4096_bf16"),
        # an fp32 training step with ragged sizes
        dict(_linear(1000, 1100, 1536, "fp32", "silu", train=True), name="linear_train_1000x1100x1536_fp32"),
        # one short answer's loss through autograd
        dict(_policy(64, 32000, "bf16", "autograd"), name="policy_64x32000_bf16"),
        # a minibatch of answers with a vocabulary of odd size, loss and gradient at once
        dict(_policy(8192, 50257, "bf16", "fused"), name="policy_8192x50257_bf16"),
        # fp32 logits with a padded vocabulary (its last columns are -inf), through autograd
        dict(_policy(1000, 32768, "fp32", "autograd", masked=0.1, pad=100), name="policy_1000x32768_fp32"),
        # the parameters that mHC adds to a model of 48 layers: 192 tensors of 4, 4, 16 and 4096 floats
        dict(_adamw(48, 4, 4096, 0, 0, "fp32"), name="adamw_48x4x4096_fp32"),
        # a bf16 model with fp32 masters and states: 16 layers with a 4096 x 4096 matrix each
        dict(_adamw(16, 4, 4096, 4096, 4096, "bf16", master=True), name="adamw_16x4096x4096_bf16"),
        # the same with states in 8 bits, ragged sizes
        dict(_adamw(24, 3, 1001, 3001, 2050, "bf16", master=True, bits=8), name="adamw_24x3001x2050_8bit"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "policy", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "linear":
        train = rng.random() < 0.5
        M = _log(rng, 1, 16384)
        N, K = (_log(rng, 256, 8192) for _ in range(2))
        if rng.random() < 0.6:  # most layers' widths are multiples of 64
            N, K = 64 * max(4, N // 64), 64 * max(4, K // 64)
        return _linear(M, N, K, dtype, rng.choice(ACTS), train, rng.random() < 0.7, rng.random() < 0.5)
    if kind == "policy":
        T, V = _log(rng, 1, 8192), _log(rng, 1000, 131072)
        T = max(1, min(T, 8192 * 50257 // (V if dtype != "fp32" else 2 * V)))
        form = rng.choice(("forward", "autograd", "fused"))
        return _policy(T, V, dtype, form, rng.choice((0.0, 0.25, 0.5)), rng.choice((0, 0, V // 50)), rng.choice((0.0, 0.05)),
                       65536.0 if dtype == "fp16" else 1.0)
    layers, n, C = _log(rng, 1, 48), rng.choice((2, 3, 4, 8, 16, 32)), _log(rng, 32, 8192)
    rows, cols = _log(rng, 16, 4096), _log(rng, 16, 4096)
    if rng.random() < 0.25:
        rows = cols = 0
    return _adamw(layers, n, C, rows, cols, dtype, dtype != "fp32" and rng.random() < 0.7, rng.choice((8, 32)))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _masked(case):
    return int(case["masked"] * case["T"])


def _sizes(case):
    n, C, matrix = case["n"], case["C"], case["rows"] * case["cols"]
    return ([n, n, n * n, C] + ([matrix] if matrix else [])) * case["layers"]


def _prepare_linear(case, g):
    M, N, K, dt = case["M"], case["N"], case["K"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"x": normal(M, K), "w": normal(N, K, scale=K ** -0.5), "b": normal(N, scale=0.5) if case["bias"] else None,
         "r": normal(M, N) if case["residual"] else None}
    if case["train"]:
        s["g"] = normal(M, N, scale=0.1)
        for k in "xwbr":
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _prepare_policy(case, g):
    T, V, dt, live = case["T"], case["V"], DTYPES[case["dtype"]], case["V"] - case["pad"]
    actions = torch.randint(0, live, (T,), generator=g, device="cuda")
    logits = torch.randn(T, V, generator=g, device="cuda").mul_(2.0)
    logits.scatter_add_(1, actions[:, None], torch.full((T, 1), 6.0, device="cuda"))  # answers are mostly likely ones
    logits[:, live:] = -math.inf
    logits = logits.to(dt)
    logp = torch.cat([torch.log_softmax(p.float(), -1).gather(1, a[:, None])[:, 0] for p, a in zip(logits.split(1024), actions.split(1024))])
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[torch.randperm(T, generator=g, device="cuda")[:_masked(case)]] = False
    s = {"logits": logits, "actions": actions, "mask": mask, "old": logp + 0.2 * torch.randn(T, generator=g, device="cuda"),
         "ref": logp + 0.3 * torch.randn(T, generator=g, device="cuda") if case["kl"] else None,
         "adv": torch.randn(T, generator=g, device="cuda")}
    if case["form"] == "autograd":
        logits.requires_grad_(True)
        s["upstream"] = torch.tensor(case["scale"], device="cuda")
    return s


def _encode(t):
    """An e4m3 code for each value of t [blocks, BLOCK], in units of a scale for each block."""
    top = t.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
    return (t * (448.0 / top)).to(torch.float8_e4m3fn), top * (1.0 / 448.0)


def _prepare_adamw(case, g):
    sizes, dt = _sizes(case), DTYPES[case["dtype"]]
    starts = [0]
    for k in sizes:
        starts.append(starts[-1] + -(-k // BLOCK) * BLOCK)
    total = starts[-1]
    inside = torch.zeros(total + 1, device="cuda")
    edges = torch.tensor([e for s, k in zip(starts, sizes) for e in (s, s + k)], device="cuda")
    signs = torch.tensor([1.0, -1.0], device="cuda").repeat(len(sizes))
    inside = inside.scatter_add_(0, edges, signs)[:total].cumsum(0)  # 1 inside a tensor, 0 in the gap after it

    def normal(scale):
        return torch.randn(total, generator=g, device="cuda").mul_(scale).mul_(inside)

    master, grad = normal(0.02), normal(1e-3)
    m, v = normal(3e-4), normal(1e-3).square_()
    s = {"p": master.to(dt), "g": grad.to(dt), "master": master if case["master"] else None}
    if case["bits"] == 32:
        s.update(m=m, v=v, scales=None)
    else:
        mc, ms = _encode(m.view(-1, BLOCK))
        rc, rs = _encode(v.sqrt().view(-1, BLOCK))
        s.update(m=mc.view(-1), v=rc.view(-1), scales=torch.cat([ms, rs], 1))

    def parts(flat):  # the tensors that a model holds, as views of a flat buffer
        return None if flat is None else [flat[a:a + k] for a, k in zip(starts, sizes)]

    s["lists"] = {k: parts(s[k]) for k in ("p", "g", "master", "m", "v")}
    s["lists"]["scales"] = None if s["scales"] is None else [
        s["scales"][a // BLOCK:(a + k + BLOCK - 1) // BLOCK] for a, k in zip(starts, sizes)]
    return s


def prepare(case, seed):
    if own:
        package = str(Path(__file__).resolve().parents[1] / "mhc-mlx_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"linear": _prepare_linear, "policy": _prepare_policy, "adamw": _prepare_adamw}[case["kind"]](case, g)
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _act(z, act):
    """act(z) and its derivative, in z's type."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).to(z.dtype)
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        p = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    c, k = (2.0 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(c * (z + k * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * k * z * z)


def _plain_linear(s, case):
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = torch.matmul(x, w.t())
    if s["b"] is not None:
        z = z + s["b"].detach().float()
    a, d = _act(z, case["act"])
    out = (a if s["r"] is None else a + s["r"].detach().float()).to(dt)
    if not case["train"]:
        return {"out": out}
    dz = s["g"].float() * d
    r = {"out": out, "dx": torch.matmul(dz, w).to(dt), "dw": torch.matmul(dz.t(), x).to(dt)}
    if s["b"] is not None:
        r["db"] = torch.matmul(torch.ones(1, dz.shape[0], device=dz.device), dz)[0].to(dt)
    if s["r"] is not None:
        r["dr"] = s["g"]
    return r


def _plain_policy(s, case):
    z, mask = s["logits"].detach().float(), s["mask"]
    T = z.shape[0]
    rows, at = torch.arange(T, device=z.device), torch.where(mask, s["actions"], 0)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logp = z[rows, at] - top[:, 0] - torch.log(total[:, 0])
    ratio, adv = torch.exp(logp - s["old"]), s["adv"]
    free, held = ratio * adv, torch.clamp(ratio, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    each = -torch.minimum(free, held)
    coef = torch.where(free <= held, -free, 0.0)
    if s["ref"] is not None:
        gap = s["ref"] - logp
        each = each + case["kl"] * (torch.exp(gap) - gap - 1.0)
        coef = coef + case["kl"] * (1.0 - torch.exp(gap))
    count = mask.sum().clamp(min=1)
    r = {"loss": torch.where(mask, each, 0.0).sum() / count, "logp": torch.where(mask, logp, 0.0)}
    if case["form"] != "forward":
        coef = torch.where(mask, coef, 0.0)[:, None] * (case["scale"] / count)
        grad = -(e / total) * coef
        grad[rows, at] += coef[:, 0]
        r["dlogits"] = torch.where(mask[:, None], grad, 0.0).to(s["logits"].dtype)
    return r


def _plain_adamw(s, case):
    b1, b2 = BETAS
    g = s["g"].float()
    p = s["p"].float() if s["master"] is None else s["master"]
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK).float() * s["scales"][:, :1]).view(-1)
        r = (v.view(-1, BLOCK).float() * s["scales"][:, 1:]).view(-1)
        v = r * r
    p = p * (1.0 - LR * DECAY)
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    r = torch.sqrt(v)
    p = p - (m / (r * (1.0 / math.sqrt(1.0 - b2 ** STEP)) + EPS)) * (LR / (1.0 - b1 ** STEP))
    if case["bits"] == 8:
        mc, ms = _encode(m.view(-1, BLOCK))
        rc, rs = _encode(r.view(-1, BLOCK))
        s["scales"].copy_(torch.cat([ms, rs], 1))
        m, v = mc.view(-1), rc.view(-1)
    s["m"].copy_(m)
    s["v"].copy_(v)
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    return {k: s[k] for k in ("p", "master", "m", "v", "scales") if s[k] is not None}


def _own_linear(s, case):
    from mhc_mlx_amd import linear_act

    if not case["train"]:
        return {"out": linear_act(s["x"], s["w"], s["b"], s["r"], activation=case["act"])}
    out = linear_act(s["x"], s["w"], s["b"], s["r"], activation=case["act"])
    names = [k for k in "xwbr" if s[k] is not None]
    grads = torch.autograd.grad(out, [s[k] for k in names], s["g"])
    return {"out": out.detach(), **{"d" + k: d for k, d in zip(names, grads)}}


def _own_policy(s, case):
    from mhc_mlx_amd import policy_loss, policy_loss_and_grad

    args = s["logits"], s["actions"], s["old"], s["adv"]
    more = {"ref_logp": s["ref"], "mask": s["mask"], "clip_low": CLIP_LOW, "clip_high": CLIP_HIGH, "kl_coef": case["kl"]}
    if case["form"] == "fused":
        loss, logp, dlogits = policy_loss_and_grad(*args, **more, grad_scale=case["scale"])
        return {"loss": loss, "logp": logp, "dlogits": dlogits}
    loss, logp = policy_loss(*args, **more)
    r = {"loss": loss.detach(), "logp": logp}
    if case["form"] == "autograd":
        r["dlogits"] = torch.autograd.grad(loss, s["logits"], s["upstream"])[0]
    return r


def _own_adamw(s, case):
    from mhc_mlx_amd import adamw_step_hip

    t = s["lists"]
    adamw_step_hip(t["p"], t["g"], t["m"], t["v"], step=STEP, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, masters=t["master"],
                   scales=t["scales"])
    return {k: s[k] for k in ("p", "master", "m", "v", "scales") if s[k] is not None}


def run(state):
    case = state["case"]
    if own:
        return {"linear": _own_linear, "policy": _own_policy, "adamw": _own_adamw}[case["kind"]](state, case)
    with torch.no_grad():
        return {"linear": _plain_linear, "policy": _plain_policy, "adamw": _plain_adamw}[case["kind"]](state, case)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "linear":
        M, N, K, e = case["M"], case["N"], case["K"], BYTES[case["dtype"]]
        inputs = M * K + N * K + N * case["bias"] + M * N * case["residual"]
        if not case["train"]:
            return {"bytes": e * (inputs + M * N), "flops": 2 * M * N * K}
        # the residual's gradient is the output's, which is read anyway
        return {"bytes": e * (inputs + 2 * M * N + M * K + N * K + N * case["bias"]), "flops": 6 * M * N * K}
    if case["kind"] == "policy":
        T, V, e = case["T"], case["V"], BYTES[case["dtype"]]
        live = T - _masked(case)
        grad = case["form"] != "forward"
        return {"bytes": e * V * (live + T * grad) + T * (1 + 8 + 4 + 4 + 4 + 4 * bool(case["kl"])), "flops": live * V * (4 + 2 * grad)}
    sizes, e = _sizes(case), BYTES[case["dtype"]]
    total, blocks = sum(sizes), sum(-(-k // BLOCK) for k in sizes)
    param = 8 + e if case["master"] else 2 * e
    states = 16 * total if case["bits"] == 32 else 4 * total + 16 * blocks
    return {"bytes": total * (e + param) + states, "flops": 14 * total}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_linear(s, case):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    z = x @ w.mT + (0.0 if s["b"] is None else s["b"].detach().double())
    act = case["act"]
    phi = torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    if act == "none":
        y, d = z, torch.ones_like(z)
    elif act == "relu":
        y, d = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    elif act == "silu":
        y, d = z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
    elif act == "gelu":
        y, d = z * torch.special.ndtr(z), torch.special.ndtr(z) + z * phi
    else:
        u = math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3)  # 0.5 (1 + tanh(u / 2)) is sigmoid(u)
        p = torch.sigmoid(u)
        y, d = z * p, p + z * p * torch.sigmoid(-u) * math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    if s["r"] is not None:
        y = y + s["r"].detach().double()
    if not case["train"]:
        return {"out": y}
    dz = d * s["g"].double()
    r = {"out": y, "dx": dz @ w, "dw": dz.mT @ x}
    if s["b"] is not None:
        r["db"] = (dz.mT @ torch.ones(len(dz), 1, dtype=dz.dtype, device=dz.device))[:, 0]
    if s["r"] is not None:
        r["dr"] = s["g"].double()
    return r


def _exact_policy(s, case):
    T, V = s["logits"].shape
    w = s["mask"].double()
    share = w / max(1.0, float(w.cpu().sum()))
    a = s["actions"][:, None]
    logp, grad = [], []
    for k in range(0, T, 1024):  # 64-bit copies of a part of the rows at a time
        z = s["logits"][k:k + 1024].detach().double()
        lse = torch.logsumexp(z, 1, keepdim=True)
        logp.append(torch.gather(z, 1, a[k:k + 1024]) - lse)
        if case["form"] != "forward":
            grad.append(torch.exp(z - lse).neg_())
    logp = torch.cat(logp)[:, 0]
    ratio, adv = torch.exp(logp - s["old"].double()), s["adv"].double()
    bound = torch.where(adv >= 0, 1.0 + CLIP_HIGH, 1.0 - CLIP_LOW)  # the side on which the clip takes hold
    inside = torch.where(adv >= 0, ratio <= bound, ratio >= bound)
    each = -adv * torch.where(inside, ratio, bound)
    slope = torch.where(inside, -adv * ratio, 0.0)
    if s["ref"] is not None:
        q = torch.exp(s["ref"].double() - logp)
        each = each + case["kl"] * (q - 1.0 - torch.log(q))
        slope = slope + case["kl"] * (1.0 - q)
    r = {"loss": (share * each).cpu().sum(), "logp": w * logp}
    if grad:
        c = (case["scale"] * share * slope)[:, None]
        grad = torch.cat(grad)
        grad = grad.scatter_add_(1, a, torch.ones_like(c)).mul_(c)
        r["dlogits"] = grad
    return r


def _exact_adamw(s, case):
    def e4m3(t):  # nearest value with 3 bits after the leading one, at least 2^-9 apart, ties to even
        step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(t / step) * step

    def coded(t):
        t = t.view(-1, BLOCK)
        unit = t.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100) / 448
        return e4m3(t / unit).view(-1), unit

    p = (s["p"] if s["master"] is None else s["master"]).double()
    m, v, g = s["m"].double(), s["v"].double(), s["g"].double()
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["scales"][:, :1].double()).view(-1)
        v = (v.view(-1, BLOCK) * s["scales"][:, 1:].double()).square().view(-1)
    b1, b2 = BETAS
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** STEP)) / (torch.sqrt(v / (1 - b2 ** STEP)) + EPS)
    scales = None
    if case["bits"] == 8:
        (m, ms), (v, vs) = coded(m), coded(torch.sqrt(v))
        scales = torch.cat([ms, vs], 1)
    r = {"p": p, "master": p, "m": m, "v": v, "scales": scales}
    return {k: x for k, x in r.items() if s[k] is not None}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"linear": _exact_linear, "policy": _exact_policy, "adamw": _exact_adamw}[case["kind"]](s, case)
