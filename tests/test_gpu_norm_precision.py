"""rms_norm where its last bits show: MX rows next to e4m3's borders."""
import pytest
import torch

from op_util import F32, mx_exact, mx_value, norm_exact
from veymoe.norm import rms_norm

pytestmark = pytest.mark.gpu


def _rows_beside_borders(width, centered):
    """(h, weight, eps): bf16 values of a row and fp32 weights whose normed products lie beside, but not on, a midpoint of
    e4m3's values (or 448 times a power of two, once in two groups), so near that their nearest float is the midpoint itself.
    eps makes mean(h^2) + eps four, exactly, in 64 bits; rows wider than 512 repeat their first 512 values."""
    times, width = max(1, width // 512), min(width, 512)
    gen = torch.Generator().manual_seed(width + centered)
    h = torch.randint(67, 96, (width,), generator=gen).double().mul(2).add(1) / 128      # 1.05 to 1.5, odd in 8 bits
    w = torch.empty(width)
    for i in range(width):
        fits = []
        while not fits:                              # the nearest weight and its neighbours, as far as they fit
            if i % 64 == 5:
                mid = 1.75                           # a group's largest value, beside 448 times a power of two
                h[i] = int(torch.randint(67, 96, (1,), generator=gen)) / 64 + 1 / 128
            else:
                mid = 1 + (2 * int(torch.randint(0, 6, (1,), generator=gen)) + 1) / 16     # between two eighths
            mid = mid if centered else mid / 2
            near = (2 * mid / h[i] - (0.0 if centered else 1.0)).float()
            for v in (near, torch.nextafter(near, torch.tensor(9.0)), torch.nextafter(near, torch.tensor(-9.0))):
                y = h[i] * (v.double() + (0.0 if centered else 1.0)) / 2
                if y != mid and y.float() == mid:
                    fits.append(v)
        w[i] = fits[int(torch.randint(0, len(fits), (1,), generator=gen))]
    eps = 4.0 - float(h.square().mean())
    assert torch.tensor(eps, dtype=torch.float32).double() == eps
    return h.bfloat16().repeat(times), w.repeat(times), eps


@pytest.mark.parametrize("centered", [True, False], ids=["weight", "one_plus_weight"])
@pytest.mark.parametrize("rows,pad", [(5, 0), (5, 3), (1100, 0), (1100, 3)])
@pytest.mark.parametrize("width", [64, 512, 2560])
def test_norm_to_mx_beside_borders(device, width, rows, pad, centered):
    """Every value and scale is the definition's: the row's factor is a half exactly, and products, with either sign, are
    held beyond fp32, so none may fall on the border's other side.  In plain fp32 about half of them would."""
    h, w, eps = _rows_beside_borders(width, centered)
    x = torch.zeros((rows, width + pad), dtype=torch.bfloat16)[:, :width]
    sign = 1 - 2 * (torch.arange(rows)[:, None] + torch.arange(width) // 3 & 1)
    x[:] = h * sign
    y = x.double() * (w.double() + (0.0 if centered else 1.0)) / 2
    q, scale = mx_exact(y)
    plain, _ = mx_exact((x.float() * ((w if centered else 1.0 + w) * 0.5)).double())
    assert (plain != q).double().mean() > 0.2                # the inputs tell the two apart
    got = rms_norm(x.to(device), w.to(device), eps=eps, one_centered=centered, quantize=True)
    mine = torch.exp2(got.scales.view(torch.uint8).cpu().double() - 127)
    assert torch.equal(mine, scale), (mine != scale).sum()
    off = got.values.cpu().float().double() != q
    assert not off.any(), (int(off.sum()), off.numel())


@pytest.mark.parametrize("centered", [True, False], ids=["weight", "one_plus_weight"])
@pytest.mark.parametrize("rows,width", [(40, 2560), (1500, 512), (7, 16384)])
def test_norm_to_mx_of_random_rows(device, rows, width, centered):
    """A value is off by half a step of e4m3 under its own scale and four half steps of fp32 (eight squares are summed in
    fp32: at most eight half steps of the sum, half of that in the root), and the scale is the definition's unless the
    group's largest value lies that near 448 times a power of two."""
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn((rows, width), generator=gen).bfloat16()
    w = (1 if centered else 0) + 0.2 * torch.randn(width, generator=gen)
    y, _, _ = norm_exact(x, w, one_centered=centered)
    got = rms_norm(x.to(device), w.to(device), one_centered=centered, quantize=True)
    mine = torch.exp2(got.scales.view(torch.uint8).cpu().double() - 127)
    err = y.abs() * 4.1 * F32
    step = torch.exp2(torch.frexp(y / mine.repeat_interleave(32, -1)).exponent.double().clamp(min=-5) - 4)
    assert ((mx_value(got) - y).abs() <= step / 2 * mine.repeat_interleave(32, -1) + err).all()
    top = y.abs().unflatten(-1, (-1, 32)).amax(-1)
    assert (top * (1 - 4.1 * F32) <= 448 * mine).all() and (top * (1 + 4.1 * F32) > 224 * mine).all()


@pytest.mark.parametrize("rows,width,pad", [(6, 64, 0), (6, 2560, 3), (1200, 512, 0), (1200, 1023, 3), (300, 16384, 0)])
def test_norm_of_fp32_rows(device, rows, width, pad):
    """h of whole numbers up to 8, whose squares' sum is exact in fp32: what is left are the roundings of the factor and of
    two products, a half step each (and 2^-48 of their products)."""
    gen = torch.Generator().manual_seed(rows + width)
    x = torch.zeros(rows, width + pad)[:, :width]
    x[:] = torch.randint(-8, 9, (rows, width), generator=gen).float()
    w = 1 + 0.2 * torch.randn(width, generator=gen)
    eps = 2.0 ** -20
    y = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps) * w.double()
    got = rms_norm(x.to(device), w.to(device), eps=eps).cpu().double()
    off = (got - y).abs() / (y.abs() * F32).clamp(min=1e-300)
    assert off.max() <= 3.001, float(off.max())
