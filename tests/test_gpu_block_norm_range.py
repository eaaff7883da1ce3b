"""block_norm of rows, scales and gates whose factors lie at the ends of fp32 or past them while the results do not."""
import pytest
import torch

from block_util import block_exact
from op_util import HALF_STEP, assert_within
from veymoe.norm import block_norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _check(x, residual, weight=None, **kw):
    got = block_norm(x, residual, weight, **kw)
    y, h, y_err, h_err = block_exact(x, residual, weight, **kw)
    h_err = h_err + 2.0 ** -148       # subnormal ones: half a step in front of a gain below two, half a step behind it
    if weight is not None:
        got, got_y = got[1], got[0]
        assert_within(got_y, y, y_err + (HALF_STEP[BF16] * (y.abs() + y_err) if x.dtype == BF16 else 0.0), "y")
    assert_within(got, h, h_err + (HALF_STEP[BF16] * (h.abs() + h_err) if residual.dtype == BF16 else 0.0), "h")


@pytest.mark.parametrize("rows,width", [(3, 128), (5, 333), (1100, 96)])
@pytest.mark.parametrize("size,scale", [(1e30, 1e-10), (1e30, 3e-20), (1e37, 1e-8), (1e-30, 1e25), (1e36, 1.0), (1e-35, 1e15)])
def test_a_rows_factor_past_fp32(device, rows, width, size, scale):
    """Rows of `size`, their norm's factor times `scale` and the row's gate: the results are normal numbers that three
    factors in fp32, one after the other, would give to a rounding each."""
    gen = torch.Generator().manual_seed(rows)
    x = (torch.randn((rows, width), generator=gen) * size).to(device)
    r, w = torch.zeros_like(x), (1 + 0.2 * torch.randn(width, generator=gen)).to(device)
    gate = (0.5 + torch.rand((rows, 1), generator=gen)).to(device)
    eps = 1e-6 if size > 1 else 0.0
    for kw in ({}, {"gate": gate}):
        _check(x, r, post_weight=w, scale=scale, eps=eps, **kw)
        _check(x.bfloat16(), r, post_weight=w, scale=scale, eps=eps, **kw)
    _check(x, r, post_weight=w, gate=gate * 1e-20, scale=1e-15, eps=eps)
    if size > 1e30:
        _check(x, r, scale=1e-30, gate=gate * 1e-10)     # no norm: scale times gate


@pytest.mark.parametrize("rows,width", [(3, 128), (5, 333), (1100, 96)])
@pytest.mark.parametrize("size", [1e38, 4e37, 1e-36, 2.0 ** -135])
def test_a_second_norm_past_fp32(device, rows, width, size):
    """Rows whose second norm's factor is subnormal or overflows fp32."""
    gen = torch.Generator().manual_seed(rows)
    r = (torch.randn((rows, width), generator=gen).clamp(-3, 3) * size).to(device)
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(device)
    x = torch.zeros_like(r)
    _check(x, r, w, eps=0.0)
    _check(x.bfloat16(), r, w, eps=0.0)


@pytest.mark.parametrize("kind", ["channel", "value"])
def test_sigmoid_gates_down_to_the_least(device, kind):
    """Gates whose sigmoid is subnormal: themselves within half a step of those (2^-150) and the sigmoid's own error."""
    rows, width = 4, 256
    g = -torch.linspace(80.0, 104.0, width)
    g = (g if kind == "channel" else g.expand(rows, width).contiguous()).to(device)
    x = torch.full((rows, width), 2.0 ** 60, device=device)
    h = block_norm(x, torch.zeros_like(x), gate=g, sigmoid_gate=True)
    s = torch.sigmoid(g.cpu().double()).expand(rows, width)
    assert_within(h, s * 2.0 ** 60, (s * 8 * 2.0 ** -24 + 2.0 ** -149) * 2.0 ** 60, kind)
