"""linear's activations of sums at the ends of fp32: results that are subnormal or just above, sums whose square overflows,
infinities; one to four rows, small tiles and large ones."""
import math

import pytest
import torch

from block_util import _activation
from op_util import F32, HALF_STEP, assert_within
from veymoe.linear import linear

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
ROWS = [1, 40, 4300]          # by matrix rows, small tiles, large tiles (of 128 by 128: 193 outputs, 128 inputs)
K, N = 128, 193


def _expected(v, name):
    """(value, relative error in half steps of fp32) in 64 bits."""
    if name == "swiglu":
        return v * torch.sigmoid(v), 16 + 2 * v.abs()
    y, _, steps = _activation(v, name)
    return y, steps


@pytest.mark.parametrize("activation", ["relu", "silu", "gelu", "gelu_tanh", "sigmoid", "swiglu"])
@pytest.mark.parametrize("rows", ROWS)
def test_sums_of_any_size(device, rows, activation):
    """Sums of one product, up to where their squares and they themselves overflow.  From 2^8 on every activation is the sum
    itself, one or zero, to a rounding each of the reciprocal, two products and the sum, or less than fp32 holds; where the
    definition has infinity times zero it is NaN."""
    sums = [2.0 ** 8, 2.0 ** 31, 2e19, 2.0 ** 64, 2.0 ** 65, 1e25, 1e38, 2.0 ** 127, 3.3895313892515355e38, math.inf]
    sums = torch.tensor(sums + [-s for s in sums]).bfloat16()
    w = torch.zeros((2 * N if activation == "swiglu" else N, K), dtype=BF16)
    w[:N, 5] = sums.repeat(N // len(sums) + 1)[:N]
    w[N:, 7] = 1.0
    x = torch.zeros((rows, K), dtype=BF16)
    x[:, 5] = x[:, 7] = 1.0
    want, _ = _expected(w[:N, 5].double().expand(rows, N), activation)
    for dtype in (FP32, BF16):
        got = linear(x.to(device), w.to(device), activation=activation, dtype=dtype)
        assert_within(got, want, 4 * F32 * want.abs() + HALF_STEP[dtype] * want.abs() + 2.0 ** -149, activation)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "sigmoid", "swiglu"])
@pytest.mark.parametrize("rows", ROWS)
def test_results_down_to_the_least(device, rows, activation):
    """Sums over which the results fall through the end of fp32's normal range to zero: a relative error, and of subnormal
    ones half a step of the last rounding."""
    low, high = {"gelu": (11.0, 14.6), "gelu_tanh": (8.5, 11.4)}.get(activation, (78.0, 110.0))
    sums = -torch.linspace(low, high, N)
    b = torch.cat([sums, torch.ones(N)]) if activation == "swiglu" else sums
    x, w = torch.zeros((rows, K), dtype=BF16), torch.zeros((len(b), K), dtype=BF16)
    want, steps = _expected(sums.double().expand(rows, N), activation)
    assert want.abs().min() < 2.0 ** -148 and want.abs().max() > 2.0 ** -120
    err = want.abs() * F32 * steps + 2.0 ** -150
    for dtype in (FP32, BF16):
        got = linear(x.to(device), w.to(device), b.to(device), activation=activation, dtype=dtype)
        assert_within(got, want, err + ((want.abs() + err) * HALF_STEP[BF16] + 2.0 ** -134 if dtype == BF16 else 0.0), activation)
