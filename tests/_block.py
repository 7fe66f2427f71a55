"""float64 references and error bounds for add_rms_norm, the int8 rows and their product, and linear_cross_entropy.

Bounds are worst cases of the formulas in fp32 (unit roundoff 2^-24) with the
roundings that the operators make, element by element, as in _train.py.
"""

import torch

from tests._train import LEAST, U32, UNIT, act64


def chain(C):
    """Additions that a term of a row's sum goes through: a thread's own, a wave's and a workgroup's."""
    return min(C, 128 + C // 1024)


def norm64(x, r, w, eps):
    """(h as stored, h in float64, 1 / rms, relative error of the operator's factor)."""
    h = x.detach() if r is None else (x.detach().float() + r.detach().float()).to(x.dtype)
    z = h.double()
    s = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
    # half the mean's error (a sum of positive terms, a division, eps), and the root's and the division's
    return h, z, s, (chain(x.shape[-1]) / 2 + 6) * U32


def ones(w, z):
    return torch.ones(z.shape[-1], dtype=torch.float64, device=z.device) if w is None else w.detach().double()


def normed64(x, r, w, eps):
    """(h, y, bound of y in x's dtype)."""
    h, z, s, off = norm64(x, r, w, eps)
    y = z * s * ones(w, z)
    return h, y, (off + 3 * U32 + 1.01 * UNIT[x.dtype]) * y.abs() + LEAST[x.dtype]


def norm_grads64(h, z, s, off, w, dy, dh, dtype, w_dtype):
    """((dx, bound), (dw, bound)) for 2-d rows."""
    C = z.shape[-1]
    wd, dy = ones(w, z), dy.double()
    n, g = z * s, dy * wd
    along = (g * n).mean(-1, keepdim=True)
    size = (g * n).abs().mean(-1, keepdim=True)
    off_n, off_along = off + U32, (off + (chain(C) + 4) * U32) * size
    dx = s * (g - n * along)
    e = s * (g.abs() * (off + 3 * U32) + n.abs() * (along.abs() * (off + off_n + 4 * U32) + off_along))
    if dh is not None:
        dx = dx + dh.double()
    t = dy * n
    dw, dsize = t.sum(0), t.abs().sum(0)
    return ((dx, e + (1.01 * UNIT[dtype] + U32) * dx.abs() + LEAST[dtype]),
            (dw, (off + (len(t) + 4) * U32) * dsize + 1.01 * UNIT[w_dtype] * dw.abs() + LEAST[w_dtype]))


def check_codes(codes, scales, v, off):
    """Codes and scales of rows whose values are v (float64), known to a factor that all of a row share and `off` of it."""
    top = v.abs().amax(-1, keepdim=True)
    q = 127 * v / torch.where(top > 0, top, 1.0)
    # a code is the nearest whole number; v and the quotient take a few roundings on the way
    assert bool(((codes.double() - q).abs() <= 0.5 + 127 * 6 * U32).all())
    want = top[..., 0] / 127
    assert bool(((scales.double() - want).abs() <= (off + 6 * U32) * want + LEAST[torch.float32]).all())


def int8_product64(rows, weight, bias, residual, act, out_dtype):
    """(out, bound)."""
    xc, wc = rows.codes.double(), weight.codes.double()
    both = rows.scales.double()[..., None] * weight.scales.double()
    # the sum's way to fp32 (of each part of a reduction), two scales, the bias and the parts' sums
    z, size = (xc @ wc.t()) * both, (xc.abs() @ wc.abs().t()) * both.abs()
    dz = 24 * U32 * size
    if bias is not None:
        z, dz = z + bias.double(), dz + 2 * U32 * bias.double().abs()
    y, _ = act64(z, act)
    bound = 1.13 * dz + 16 * U32 * (z.abs() + 1)
    if act != "none":  # (as linear_act's activations of 16-bit operands are formed)
        bound = bound + 2.0 ** -21 * z.abs() + 2.0 ** -15 * y.abs()
    if residual is not None:
        y = y + residual.double()
    return y, bound + (UNIT[out_dtype] + 2 * U32) * y.abs() + LEAST[out_dtype]


def ce64(x, w, targets, weights=None, den=None, ignore_index=-100, scale=1.0):
    """A dict of (value, bound): loss, logp, dx, dw, for 2-d x."""
    dt = x.dtype
    T, V, C = len(x), len(w), x.shape[1]
    m = torch.ones(T, dtype=torch.float64, device=x.device) if weights is None else weights.double()
    m = torch.where(targets == ignore_index, 0.0, m)
    on = m != 0
    xd, wd = torch.where(on[:, None], x.detach().double(), 0.0), w.detach().double()
    y = torch.where(on, targets, 0).long()[:, None]
    z, dz = xd @ wd.t(), (C + 2) * U32 * (xd.abs() @ wd.abs().t())
    lse = torch.logsumexp(z, 1, keepdim=True)
    # a weighted mean of the logits' errors, and exponentials, their arguments (up to log V in the mean) and sums of positive terms
    off_lse = dz.amax(1, keepdim=True) + 200 * U32
    logp = torch.where(on, (z - lse).gather(1, y)[:, 0], 0.0)
    off_logp = torch.where(on, dz.gather(1, y)[:, 0] + off_lse[:, 0] + 2 * U32 * logp.abs(), 0.0)
    D = den or float(m.sum()) or 1.0
    loss, off_loss = -(m * logp).sum() / D, (m.abs() * off_logp).sum() / abs(D)
    r = {"loss": (loss, off_loss + 8 * U32 * (m * logp).abs().sum() / abs(D)), "logp": (logp, off_logp)}
    p = torch.exp(z - lse)
    top = float(m.abs().max()) or 1.0
    c = (m / top)[:, None]
    d = p.scatter_add(1, y, torch.full_like(lse, -1.0)) * c
    unit = 2.0 ** 14 if dt == torch.float16 else 1.0
    off = c.abs() * p * (dz + off_lse + (16 + 3 * (z - lse).abs()) * U32) + 4 * U32 * d.abs()
    off = off + 1.01 * UNIT[dt] * d.abs() + LEAST[dt] / unit
    f = scale * top / D
    for name, got, size, e, terms in (("dx", d @ wd, d.abs() @ wd.abs(), off @ wd.abs(), V), ("dw", d.t() @ xd, d.abs().t() @ xd.abs(), off.t() @ xd.abs(), T)):
        r[name] = (f * got, abs(f) * (1.02 * e + (terms + 8) * U32 * size) + UNIT[dt] * (f * got).abs() + LEAST[dt])
    return r
