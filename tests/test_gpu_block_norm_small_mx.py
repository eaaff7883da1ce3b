"""block_norm to MX of rows that a small gain takes to the ends of fp32 and past them: e4m3's is their one rounding there too."""
import pytest
import torch

from block_util import block_exact
from op_util import mx_exact, mx_value
from veymoe.norm import block_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-90, -100, -104, -112, -118, -121, -124, -127, -130, -136, -140])
@pytest.mark.parametrize("rows,width", [(40, 2560), (1500, 512)])
def test_values_down_to_the_least(device, rows, width, power):
    """Values around 2^power: the definition's themselves, of the 64-bit values."""
    gen = torch.Generator().manual_seed(rows - power)
    x, r = torch.randn((2, rows, width), generator=gen)
    w = (1 + 0.2 * torch.randn(width, generator=gen)) * 2.0 ** max(power, -126)
    if power < -126:                                    # past fp32's normal gains: rows of which one value is large
        x[:, 0] = 2.0 ** (-126 - power) * width ** 0.5
        w = w.clone()
        w[0] = 0.0
    x, r, w = x.to(device), 0.5 * r.to(device), w.to(device)
    got, _ = block_norm(x, r, w, quantize=True)
    y, _, _, _ = block_exact(x, r, w)
    values, scales = mx_exact(y)
    mine, want = mx_value(got), values * scales.repeat_interleave(32, -1)
    assert torch.equal(mine, want), (int((mine != want).sum()), mine.numel())
