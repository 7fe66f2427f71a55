"""The operators between the residual stream and a model's answer, on one GPU: what is measured of them, and their plain forms.

Three kinds of case, one for each operator:

  norm   add_rms_norm / add_rms_norm_int8: RMS norm with the residual's addition; its output in the input's type, with its
         gradients, or in int8 with a scale for each row
  int8   linear_int8: a product of int8 rows with scales for each token and channel, from rows that are there, from 16-bit
         activations (quantize_int8) or behind the norm (add_rms_norm_int8)
  ce     linear_cross_entropy / linear_cross_entropy_and_grad: softmax cross entropy over a vocabulary from the last hidden states
         and the head's weight

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
EPS = 1e-6


def _norm(T, C, dtype, form, residual=True, weight="same"):
    return {"kind": "norm", "T": T, "C": C, "dtype": dtype, "form": form, "residual": residual, "weight": weight}


def _int8(M, N, K, dtype, source, act="none", bias=True, residual=False):
    return {"kind": "int8", "M": M, "N": N, "K": K, "dtype": dtype, "source": source, "act": act, "bias": bias, "residual": residual}


def _ce(T, V, C, dtype, form, masked=0.25, scale=1.0):
    return {"kind": "ce", "T": T, "V": V, "C": C, "dtype": dtype, "form": form, "masked": masked, "scale": scale}


def listed():
    return [
        # one token between two layers of a block: latency counts
        dict(_norm(1, 4096, "bf16", "forward"), name="norm_1x4096_bf16"),
        # a decoding step of a batch before a product in 8 bits
        dict(_norm(64, 4096, "bf16", "int8"), name="norm_int8_64x4096_bf16"),
        # a training step's call between two layers, with the gradients of both of its outputs; the weight is an fp32 parameter
        dict(_norm(8192, 4096, "bf16", "train", weight="fp32"), name="norm_train_8192x4096_bf16"),
        # an fp32 training step with ragged sizes
        dict(_norm(1001, 1100, "fp32", "train"), name="norm_train_1001x1100_fp32"),
        # one token's activations through a square layer in 8 bits
        dict(_int8(1, 4096, 4096, "bf16", "activations", "gelu"), name="int8_1x4096x4096_bf16"),
        # a decoding step of a small batch through the widening product of a feed-forward block
        dict(_int8(32, 8192, 2048, "fp16", "rows", "silu"), name="int8_32x8192x2048_fp16"),
        # a prompt of odd length at widths that are no multiple of a vector
        dict(_int8(1001, 2050, 1100, "bf16", "rows", "relu", residual=True), name="int8_1001x2050x1100_bf16"),
        # the norm and the product behind it, as a block has them: a prompt of 2048 tokens
        dict(_int8(2048, 8192, 4096, "bf16", "norm", "gelu_tanh"), name="int8_norm_2048x8192x4096_bf16"),
        # prefill of a large batch through the widening product
        dict(_int8(16384, 16384, 4096, "bf16", "rows", bias=False), name="int8_16384x16384x4096_bf16"),
        # the log probabilities of one short answer, without gradients
        dict(_ce(64, 32000, 2048, "bf16", "forward"), name="ce_64x32000x2048_bf16"),
        # a training step's loss of 8192 tokens over a vocabulary of odd size, a quarter of them a prompt's
        dict(_ce(8192, 50257, 4096, "bf16", "fused"), name="ce_train_8192x50257x4096_bf16"),
        # an fp32 model's loss through autograd
        dict(_ce(1000, 32768, 1024, "fp32", "autograd", masked=0.1), name="ce_train_1000x32768x1024_fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "int8", "ce"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    even = rng.random() < 0.6  # most models' widths are multiples of 64

    def width(low, high):
        n = _log(rng, low, high)
        return 64 * max(low // 64, n // 64) if even else n

    if kind == "norm":
        form = rng.choice(("forward", "train", "int8"))
        if form == "int8" and dtype == "fp32":
            dtype = "bf16"
        T, C = _log(rng, 1, 16384), width(64, 16384)
        T = max(1, min(T, 8192 * 4096 * 2 // (C * BYTES[dtype])))
        return _norm(T, C, dtype, form, rng.random() < 0.8, rng.choice(("same", "fp32")) if form != "int8" else "same")
    if kind == "int8":
        source = rng.choice(("rows", "rows", "activations", "norm"))
        if source != "rows" and dtype == "fp32":
            dtype = "bf16"
        M, N, K = _log(rng, 1, 16384), width(256, 16384), width(256, 8192)
        return _int8(M, N, K, dtype, source, rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.4)
    T, V, C = _log(rng, 1, 8192), _log(rng, 1000, 131072), width(256, 4096)
    T = max(1, min(T, int(8192 * 50257 * 4096 // (V * C * (8 if dtype == "fp32" else 1)))))
    form = rng.choice(("forward", "autograd", "fused"))
    return _ce(T, V, C, dtype, form, rng.choice((0.0, 0.25, 0.5)), 65536.0 if dtype == "fp16" else 1.0)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _masked(case):
    return int(case["masked"] * case["T"])


def _rows_of_codes(t):
    """int8 codes of t's rows and a scale for each."""
    top = t.abs().amax(1).clamp(min=2.0 ** -100)
    return torch.round(t * (127.0 / top)[:, None]).to(torch.int8), top * (1.0 / 127.0)


def _prepare_norm(case, g):
    T, C, dt = case["T"], case["C"], DTYPES[case["dtype"]]
    wt = torch.float32 if case["weight"] == "fp32" else dt

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"x": normal(T, C), "r": normal(T, C, scale=2.0) if case["residual"] else None,
         "w": (1.0 + 0.1 * torch.randn(C, generator=g, device="cuda")).to(wt)}
    if case["form"] == "train":
        s["gy"], s["gh"] = normal(T, C, scale=0.1), normal(T, C, scale=0.1) if case["residual"] else None
        for k in "xrw":
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


def _prepare_int8(case, g):
    M, N, K, dt = case["M"], case["N"], case["K"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    s = {"b": normal(N, scale=0.5) if case["bias"] else None, "r": normal(M, N).to(dt) if case["residual"] else None}
    s["wc"], s["ws"] = _rows_of_codes(normal(N, K, scale=K ** -0.5))
    x = normal(M, K)
    if case["source"] == "rows":
        s["xc"], s["xs"] = _rows_of_codes(x)
    else:
        s["x"] = x.to(dt)
    if case["source"] == "norm":
        s["h"], s["nw"] = normal(M, K, scale=2.0).to(dt), (1.0 + 0.1 * normal(K)).to(dt)
    return s


def _prepare_ce(case, g):
    T, V, C, dt = case["T"], case["V"], case["C"], DTYPES[case["dtype"]]
    w = torch.randn(V, C, generator=g, device="cuda").mul_(1.3 * C ** -0.5).to(dt)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    x = torch.randn(T, C, generator=g, device="cuda").add_(w[y].float(), alpha=4.0).to(dt)  # targets are mostly likely ones
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[torch.randperm(T, generator=g, device="cuda")[:_masked(case)]] = False
    s = {"x": x, "w": w, "y": y, "mask": mask}
    if case["form"] == "autograd":
        x.requires_grad_(True)
        w.requires_grad_(True)
        s["upstream"] = torch.tensor(case["scale"], device="cuda")
    return s


def prepare(case, seed):
    if own:
        package = str(Path(__file__).resolve().parents[1] / "mhc-mlx_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"norm": _prepare_norm, "int8": _prepare_int8, "ce": _prepare_ce}[case["kind"]](case, g)
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return z * (0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z


def _plain_normed(x, r, w):
    """The sum in x's type, and in fp32: the sum, the norm's factor and the normed rows."""
    h = x.detach() if r is None else (x.detach().float() + r.detach().float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    return h, hf, rstd, hf * rstd * w.detach().float()


def _plain_codes(y):
    """Codes (as floats) and scales of rows."""
    scale = y.abs().amax(1, keepdim=True) * (1.0 / 127.0)
    return torch.round(y / scale.clamp(min=2.0 ** -120)), scale


def _plain_norm(s, case):
    h, hf, rstd, y = _plain_normed(s["x"], s["r"], s["w"])
    r = {} if s["r"] is None else {"h": h}
    if case["form"] == "int8":
        codes, scale = _plain_codes(y)
        return {**r, "values": (codes * scale).to(h.dtype), "scales": scale[:, 0]}
    r["y"] = y.to(h.dtype)
    if case["form"] == "train":
        gy = s["gy"].float()
        g = gy * s["w"].detach().float()
        d = rstd * (g - hf * (rstd * rstd * (g * hf).mean(1, keepdim=True)))
        if s["gh"] is not None:
            d = d + s["gh"].float()
        r["dx"] = d.to(h.dtype)
        if s["r"] is not None:
            r["dr"] = r["dx"]
        r["dw"] = torch.matmul(torch.ones(1, len(hf), device=hf.device), gy * hf * rstd)[0].to(s["w"].dtype)
    return r


def _plain_int8(s, case):
    r = {}
    if case["source"] == "rows":
        xc, xs = s["xc"].float(), s["xs"][:, None]
    elif case["source"] == "activations":
        xc, xs = _plain_codes(s["x"].float())
    else:
        r["h"], _, _, y = _plain_normed(s["x"], s["h"], s["nw"])
        xc, xs = _plain_codes(y)
    z = torch.matmul(xc, s["wc"].float().t()) * xs * s["ws"]
    if s["b"] is not None:
        z = z + s["b"]
    z = _act(z, case["act"])
    if s["r"] is not None:
        z = z + s["r"].float()
    return {**r, "out": z.to(DTYPES[case["dtype"]])}


def _plain_ce(s, case):
    x, w, y, mask = s["x"].detach().float(), s["w"].detach().float(), s["y"], s["mask"]
    rows = torch.arange(len(y), device=y.device)
    z = torch.matmul(x, w.t())
    top = z.amax(1, keepdim=True)
    at = z[rows, y] - top[:, 0]
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logp = torch.where(mask, at - torch.log(total[:, 0]), 0.0)
    count = mask.sum().clamp(min=1)
    r = {"loss": -logp.sum() / count, "logp": logp}
    if case["form"] != "forward":
        each = torch.where(mask, case["scale"] / count, 0.0)
        d = e * (each[:, None] / total)
        d[rows, y] -= each
        r["dx"] = torch.matmul(d, w).to(s["x"].dtype)
        r["dw"] = torch.matmul(d.t(), x).to(s["w"].dtype)
    return r


def _own_norm(s, case):
    from mhc_mlx_amd import add_rms_norm, add_rms_norm_int8

    if case["form"] == "int8":
        rows, h = add_rms_norm_int8(s["x"], s["r"], s["w"], eps=EPS)
        r = {"values": rows.dequantize(s["x"].dtype), "scales": rows.scales}
    else:
        y, h = add_rms_norm(s["x"], s["r"], s["w"], eps=EPS)
        r = {"y": y.detach()}
    if s["r"] is not None:
        r["h"] = h.detach()
    if case["form"] == "train":
        names = [k for k in "xrw" if s[k] is not None]
        outs, grads = ([y], [s["gy"]]) if s["r"] is None else ([y, h], [s["gy"], s["gh"]])
        r.update(zip(["d" + k for k in names], torch.autograd.grad(outs, [s[k] for k in names], grads)))
    return r


def _own_int8(s, case):
    from mhc_mlx_amd import Int8Rows, add_rms_norm_int8, linear_int8, quantize_int8

    r = {}
    if case["source"] == "rows":
        rows = Int8Rows(s["xc"], s["xs"])
    elif case["source"] == "activations":
        rows = quantize_int8(s["x"])
    else:
        rows, r["h"] = add_rms_norm_int8(s["x"], s["h"], s["nw"], eps=EPS)
    r["out"] = linear_int8(rows, Int8Rows(s["wc"], s["ws"]), s["b"], s["r"], activation=case["act"], output_dtype=DTYPES[case["dtype"]])
    return r


def _own_ce(s, case):
    from mhc_mlx_amd import linear_cross_entropy, linear_cross_entropy_and_grad

    if case["form"] == "fused":
        loss, logp, dx, dw = linear_cross_entropy_and_grad(s["x"], s["w"], s["y"], mask=s["mask"], grad_scale=case["scale"])
        return {"loss": loss, "logp": logp, "dx": dx, "dw": dw}
    loss, logp = linear_cross_entropy(s["x"], s["w"], s["y"], mask=s["mask"])
    r = {"loss": loss.detach(), "logp": logp}
    if case["form"] == "autograd":
        r["dx"], r["dw"] = torch.autograd.grad(loss, [s["x"], s["w"]], s["upstream"])
    return r


def run(state):
    case = state["case"]
    if own:
        return {"norm": _own_norm, "int8": _own_int8, "ce": _own_ce}[case["kind"]](state, case)
    with torch.no_grad():
        return {"norm": _plain_norm, "int8": _plain_int8, "ce": _plain_ce}[case["kind"]](state, case)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        T, C, r = case["T"], case["C"], int(case["residual"])
        we = e if case["weight"] == "same" else 4
        if case["form"] == "int8":
            # the codes are read once more and written as the values that they stand for
            return {"bytes": T * C * (e * (1 + 2 * r) + 1 + 1 + e) + 4 * T + we * C, "flops": 10 * T * C}
        if case["form"] == "forward":
            return {"bytes": e * T * C * (2 + 2 * r) + we * C, "flops": 5 * T * C}
        # the sum is read again for the gradient, with those of the outputs; the gradients of both inputs are one tensor
        return {"bytes": e * T * C * (2 + 2 * r + 3 + r) + 2 * we * C, "flops": 15 * T * C}
    if case["kind"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        rows = {"rows": M * K + 4 * M, "activations": e * M * K, "norm": 3 * e * M * K + e * K}[case["source"]]
        return {"bytes": rows + N * K + 4 * N + 4 * N * case["bias"] + e * M * N * (1 + case["residual"]), "flops": 2 * M * N * K}
    T, V, C = case["T"], case["V"], case["C"]
    live = T - _masked(case)
    grad = case["form"] != "forward"
    return {"bytes": e * C * ((live + V) + (T + V) * grad) + T * (1 + 8 + 4), "flops": live * V * C * (6 if grad else 2)}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_sum(x, r):
    """x + r, rounded once to their type: what the operator hands on is what it norms."""
    x = x.detach()
    return x.double() if r is None else (x.double() + r.detach().double()).to(x.dtype).double()


def _exact_rows(v):
    """The values that v's rows are held as, and their scales."""
    scales = v.abs().max(dim=1).values / 127
    units = torch.where(scales > 0, scales, 1.0)[:, None]
    return torch.round(v / units) * units, scales


def _exact_norm(s, case):
    h, w = _exact_sum(s["x"], s["r"]), s["w"].detach().double()
    C = h.shape[1]
    length = torch.sqrt(h.square().sum(1, keepdim=True) / C + EPS)
    n = h / length
    r = {} if s["r"] is None else {"h": h}
    if case["form"] == "int8":
        r["values"], r["scales"] = _exact_rows(n * w)
        return r
    r["y"] = n * w
    if case["form"] == "train":
        gy = s["gy"].double()
        along = (gy * w * n).sum(1, keepdim=True) / C
        r["dx"] = (gy * w - n * along) / length + (0.0 if s["gh"] is None else s["gh"].double())
        if s["r"] is not None:
            r["dr"] = r["dx"]
        r["dw"] = (n * gy).cpu().sum(0)
    return r


def _exact_int8(s, case):
    r = {}
    if case["source"] == "rows":
        x = s["xc"].double() * s["xs"].double()[:, None]
    elif case["source"] == "activations":
        x = _exact_rows(s["x"].double())[0]
    else:
        r["h"] = _exact_sum(s["x"], s["h"])
        y = r["h"] / torch.sqrt(r["h"].square().sum(1, keepdim=True) / r["h"].shape[1] + EPS) * s["nw"].double()
        x = _exact_rows(y)[0]
    z = x @ (s["wc"].double() * s["ws"].double()[:, None]).mT
    if s["b"] is not None:
        z += s["b"].double()
    act = case["act"]
    if act == "relu":
        z = torch.where(z > 0, z, 0.0)
    elif act == "silu":
        z = z * torch.sigmoid(z)
    elif act == "gelu":
        z = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":
        z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))  # 0.5 (1 + tanh(u / 2)) is sigmoid(u)
    if s["r"] is not None:
        z = z + s["r"].double()
    return {**r, "out": z}


def _exact_ce(s, case):
    x, w, y = s["x"].detach(), s["w"].detach().double(), s["y"][:, None]
    m = s["mask"].double()
    share = m / max(1.0, float(m.cpu().sum()))
    logp, dx, dw = [], [], 0.0
    for k in range(0, len(x), 2048):  # 64-bit logits of a part of the rows at a time
        xk, yk = x[k:k + 2048].double(), y[k:k + 2048]
        z = xk @ w.mT
        lse = torch.logsumexp(z, 1, keepdim=True)
        logp.append(torch.gather(z, 1, yk) - lse)
        if case["form"] != "forward":
            c = (case["scale"] * share[k:k + 2048])[:, None]
            d = z.sub_(lse).exp_().scatter_add_(1, yk, torch.full_like(lse, -1.0)).mul_(c)
            dx.append(d @ w)
            dw = dw + d.mT.contiguous() @ xk
    logp = torch.cat(logp)[:, 0]
    r = {"loss": -(share * logp).cpu().sum(), "logp": m * logp}
    if dx:
        r["dx"], r["dw"] = torch.cat(dx), dw
    return r


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "int8": _exact_int8, "ce": _exact_ce}[case["kind"]](s, case)
