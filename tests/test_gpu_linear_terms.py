"""linear's sums where a few lost bits show: terms that cancel, in neighbouring inputs too, and inputs below bf16's normal
range; by matrix rows, small tiles and large ones."""
import pytest
import torch

from op_util import HALF_STEP, assert_within, mx_value
from veymoe.linear import linear
from veymoe.norm import mx_quantize

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
ROWS = [1, 2, 4, 40, 4300]


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("apart", [1, 2, 3, 17])
@pytest.mark.parametrize("rows", ROWS)
def test_terms_that_cancel(device, rows, apart, mx):
    """Every 32 inputs hold 256, `apart` inputs on -256, and before, behind or between them m 2^-9, m up to 3, by ones of
    either sign: sums of whole multiples of 2^-9 below 2^15, exact in fp32 in any order."""
    k, n = 256, 193
    m = (torch.arange(rows) % 3 + 1).float()
    sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    w = sign[:, None].expand(n, k).bfloat16().contiguous().to(device)
    want = (m[:, None] * (k // 32) * 2.0 ** -9 * sign).to(device)
    for first in (0, 1, 6, 7):
        for small in (first - 1, first + apart + 1, first + (apart + 1) // 2 if apart > 1 else 30):
            x = torch.zeros((rows, k // 32, 32))
            x[:, :, first], x[:, :, first + apart] = 256.0, -256.0
            x[:, :, small % 32] = m[:, None] * 2.0 ** -9
            x = x.view(rows, k).bfloat16().to(device)
            a, b = (mx_quantize(x), mx_quantize(w)) if mx else (x, w)
            assert not mx or torch.equal(a.dequantize(BF16), x)
            assert torch.equal(linear(a, b, dtype=FP32), want), (first, small)


@pytest.mark.parametrize("rows", ROWS)
def test_bf16_below_the_normal_range(device, rows):
    """Subnormal inputs on either side: one product to an output, exact in fp32."""
    k, n = 128, 193
    x, w = torch.zeros((rows, k)), torch.zeros((n, k))
    j = torch.arange(n) % 7 + 1
    x[:, 0], x[:, 1] = 2.0 ** -133, 2.0 ** 100
    x[:, 70] = 1.5 * 2.0 ** -128
    w[:, 0] = j * 2.0 ** 100                     # j 2^-33
    w[:, 1] = j * 2.0 ** -133                    # j 2^-33
    w[:, 70] = 2.0 ** 96                         # 1.5 2^-32
    want = (2 * j * 2.0 ** -33 + 1.5 * 2.0 ** -32).float().expand(rows, n).to(device)
    assert torch.equal(linear(x.bfloat16().to(device), w.bfloat16().to(device), dtype=FP32), want)


@pytest.mark.parametrize("rows", ROWS)
def test_mx_below_bf16s_normal_range(device, rows):
    """Scales far apart cancel in the product.  Below bf16's normal range values are rounded to multiples of 2^-133: off by
    2^-134 at most, times the matrix value."""
    x, w = torch.full((rows, 128), 1e-30), torch.full((193, 128), 1e30)
    x[:, 32:] = 0
    x[0] = 1e-40
    x[rows // 2, 40] = 1e-37
    xq, wq = mx_quantize(x.to(device)), mx_quantize(w.to(device))
    xv, wv = mx_value(xq), mx_value(wq)
    want = xv @ wv.T
    err = (xv != 0).double() @ wv.abs().T * 2.0 ** -134 + 129 * 2 * 2.0 ** -24 * want.abs()
    for dtype in (FP32, BF16):
        got = linear(xq, wq, dtype=dtype)
        assert_within(got, want, err + (want.abs() + err) * HALF_STEP[dtype])
    # multiples of 2^-133 are kept as they are: one of them by powers of two, a group each
    x = torch.zeros((rows, 128))
    x[:, 3], x[:, 33], x[:, 101] = 2.0 ** -133, 3 * 2.0 ** -133, 2.0 ** -127
    w = torch.zeros((193, 128))
    w[:, 3], w[:, 33], w[:, 101] = 2.0 ** 100, 2.0 ** 101, 2.0 ** 95
    want = 2.0 ** -33 + 3 * 2.0 ** -32 + 2.0 ** -32
    assert (linear(mx_quantize(x.to(device)), mx_quantize(w.to(device)), dtype=FP32) == want).all()
