"""float64 references and error bounds for linear_act, the policy loss and AdamW.

Bounds are worst cases of the formulas in fp32 (unit roundoff 2^-24) with the
roundings that the operators make, element by element.
"""

import math

import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # unit roundoffs: 24, 8, 11 bits
LEAST = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half the least subnormal


def act64(z, act):
    """act(z) and act'(z) in float64."""
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * phi
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    c = math.sqrt(8 / math.pi)
    p = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return z * p, p + z * p * (1 - p) * c * (1 + 0.134145 * z ** 2)


def linear64(x, w, b, r, act, out_dtype):
    """(out, bound, z, act'(z), bound of z) for 2-d x, in float64."""
    x, w = x.detach().double(), w.detach().double()
    K = x.shape[1]
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.detach().double(), size + b.detach().double().abs()
    dz = (K + 2) * U32 * size
    y, d = act64(z, act)
    # the functions: a few roundings of arguments up to |z| and of the result (a slope of at most 1.13)
    bound = 1.13 * dz + 16 * U32 * (z.abs() + 1)
    if r is not None:
        y = y + r.detach().double()
    bound = bound + (UNIT[out_dtype] + 2 * U32) * y.abs() + LEAST[out_dtype]
    return y, bound, z, d, dz


def linear_grads64(x, w, g, d, dz, dtype, has_act):
    """((dx, bound), (dw, bound), (db, bound)): dz is rounded to dtype, act' to 2^-15 steps (fp32 for fp32)."""
    x, w, g = x.detach().double(), w.detach().double(), g.double()
    t = g * d
    # |act''| <= 1; act' takes a few roundings of values up to 2
    off = g.abs() * (dz + 32 * U32) + t.abs() * 4 * U32
    if has_act:
        off = off + (t.abs() * U32 if dtype == torch.float32 else g.abs() * 2.0 ** -16)
    sum_off = off
    off = off + t.abs() * 1.01 * UNIT[dtype] + LEAST[dtype]
    M, N = t.shape

    def bound(ref, size, terms, e):
        return ref, e + terms * U32 * size + UNIT[dtype] * ref.abs() + LEAST[dtype]

    one = torch.ones(1, M, dtype=torch.float64, device=x.device)
    return (bound(t @ w, t.abs() @ w.abs(), N + 2, 1.01 * off @ w.abs()),
            bound(t.t() @ x, t.abs().t() @ x.abs(), M + 2, 1.01 * off.t() @ x.abs()),
            bound((one @ t)[0], (one @ t.abs())[0], M + 2, (one @ sum_off)[0]))


def close(got, ref, bound, what=""):
    got = got.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - ref).abs() / bound).nan_to_num(math.inf).max()):.3g} bounds"


def policy64(logits, actions, old, adv, ref=None, weights=None, lo=0.2, hi=0.2, kl=0.0, den=None):
    """(loss, logp, coef) in float64: coef is w dL / dlp / D of each token, 0 where w is 0."""
    z = logits.detach().double()
    T = z.shape[0]
    w = torch.ones(T, dtype=torch.float64, device=z.device) if weights is None else weights.double()
    on = w != 0
    a = torch.where(on, actions, 0).long()
    lp = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    r, A = torch.exp(lp - old.double()), adv.double()
    free, held = r * A, r.clamp(1 - lo, 1 + hi) * A
    L, c = -torch.minimum(free, held), torch.where(free <= held, -free, 0.0)
    if ref is not None:
        gap = ref.double() - lp
        L, c = L + kl * (torch.expm1(gap) - gap), c - kl * torch.expm1(gap)
    D = den or float(w.cpu().sum()) or 1.0
    off = torch.zeros_like(L)
    return (torch.where(on, w * L, off).cpu().sum().to(z.device) / D, torch.where(on, lp, off), torch.where(on, w * c / D, off))
