"""add_rms_norm_int8: codes next to the middle between two of them."""

import pytest
import torch

from mhc_mlx_amd import add_rms_norm_int8

pytestmark = pytest.mark.gpu


def near_ties(top, each=8):
    """fp16 mantissa pairs (h, w in [1024, 2048)) and exponents whose h w is next to (k + 1/2) / 127 of top, for each k."""
    m = torch.arange(1024, 2048, dtype=torch.float64)
    h, w, e = [], [], []
    for k in range(127):
        at, shift = (2 * k + 1) * top / 254, 0
        while at < 2 ** 21:
            at, shift = at * 2, shift - 1
        for a, s in ((at, shift), (at * 2, shift - 1), (at / 2, shift + 1)):
            other = torch.floor(a / m)
            for o in (other, other + 1):
                fits = (o >= 1024) & (o < 2048)
                off = torch.where(fits, (m * o / a - 1).abs(), 9.0)
                for i in off.argsort()[:each].tolist():
                    if fits[i]:
                        h.append(float(m[i])), w.append(float(o[i])), e.append(s)
    return torch.tensor(h), torch.tensor(w), torch.tensor(e, dtype=torch.float32)


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("a,b", [(2047, 2047), (1025, 1663), (1409, 1999), (1024, 1024), (1741, 1979)])
def test_fp16_codes_next_to_ties(a, b, long):
    h, w, e = near_ties(a * b)
    x = torch.cat([torch.tensor([float(a)]), h * 2.0 ** e]) / 1024
    w = torch.cat([torch.tensor([float(b)]), w]) / 1024
    if long:  # (rows that no workgroup holds)
        x, w = (t.repeat(40000 // len(t) + 1) for t in (x, w))
    xh, wh = x.half(), w.half()
    assert torch.equal(xh.float(), x) and torch.equal(wh.float(), w)
    p = xh.double() * wh.double()
    q = 127 * p / p.max()  # (in fp64 127 p is exact, and quotients that are no ties lie further from them than a rounding)
    x = torch.stack([xh, -xh, xh.flip(0)]).cuda()
    codes = torch.stack([add_rms_norm_int8(r[None], None, v)[0].codes[0] for r, v in zip(x, (wh.cuda(), wh.cuda(), wh.flip(0).cuda()))]).cpu().double()
    want = torch.round(q)
    assert int(((q - q.floor() - 0.5).abs() < 2.0 ** -15).sum()) > 100
    assert torch.equal(codes[0], want) and torch.equal(codes[1], -want) and torch.equal(codes[2], want.flip(0))
