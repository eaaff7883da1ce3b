"""grouped_matmul where a few lost bits show: gates far below zero, and terms that cancel."""
import pytest
import torch

from op_util import F32, HALF_STEP, assert_mx_within, assert_within, mx_value
from veymoe.norm import MxTensor, mx_quantize
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("quantize", [False, True], ids=["to_bf16", "to_mx"])
@pytest.mark.parametrize("tokens", [3, 70, 300])
def test_swiglu_of_gates_far_below_zero(device, tokens, quantize, mx):
    """Gates down to -172 beside an up of up to 2^120: silu alone is below fp32's normal range from -87 on, the results are
    around one down to gates of -83 and normal down to the last.  Gate and up are exact sums of one or two terms, so silu's
    own error is all there is: 16 + 2 |g| half steps of fp32 at most."""
    n, k = 64, 64
    gates = torch.cat([torch.tensor([2.0, 1.25, 0.375, -0.375, -1.25, -2.0]), -torch.arange(81.0, 104.0),
                       -torch.arange(104.0, 174.0, 2.0)])
    coarse = (gates / 16).trunc() * 16                               # both parts exact in e4m3's four bits
    up = torch.exp2((gates.abs() * 1.4427).round().clamp(max=120))
    w = torch.zeros(2, 2 * n, k)
    w[:, :n, 0], w[:, :n, 32] = coarse, gates - coarse
    w[0, n:, 1], w[1, n:, 1] = up, -up
    x = torch.zeros(tokens, k)
    x[:, 0], x[:, 32] = 1, 1
    x[:, 1] = 0.5 + (torch.arange(tokens) % 5) * 0.125
    inds = (torch.arange(tokens) % 2).int().reshape(-1, 1)
    g = gates.double().expand(tokens, n)
    u = up.double() * x[:, 1:2].double() * torch.where(inds == 0, 1.0, -1.0).double()
    x, w = x.bfloat16().to(device), w.bfloat16().to(device)
    if mx:
        x, w = mx_quantize(x), mx_quantize(w)
        assert torch.equal(mx_value(w)[0, :n, 0] + mx_value(w)[0, :n, 32], g[0])
    want = g * torch.sigmoid(g) * u
    err = want.abs() * F32 * (16 + 2 * g.abs())
    got = grouped_matmul(x, w, inds.to(device), activation="swiglu", quantize=quantize)
    if quantize:
        assert_mx_within(MxTensor(*(t.view(tokens, -1) for t in got)), want, err)
    else:
        assert_within(got.view(tokens, n), want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [3, 70, 300, 2500])
@pytest.mark.parametrize("k", [32, 96, 256, 2560])
def test_terms_that_cancel(device, k, tokens, mx):
    """Every group of 32 holds 256, -256 and m 2^-9, m up to 3, and the matrix ones of either sign: sums of whole multiples of
    2^-9 below 2^15, exact in fp32 in any order, and m 2^-9 times the groups (up to 80), exact in bf16.  A product that drops
    what is below 2^-16 of a group's largest term finds nothing."""
    n, experts = 40, 3
    m = (torch.arange(tokens) % 3 + 1).float()
    gen = torch.Generator().manual_seed(k + tokens)
    x = torch.zeros(tokens, k // 32, 32)
    at = torch.rand((tokens, k // 32, 32), generator=gen).argsort(-1)[..., :3]
    x.scatter_(2, at, torch.stack([torch.full_like(m, 256), torch.full_like(m, -256), m * 2.0 ** -9], -1)[:, None].expand_as(at))
    sign = torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)
    w = sign[:, None].expand(experts, n, k)
    x, w = x.view(tokens, k).bfloat16().to(device), w.bfloat16().contiguous().to(device)
    if mx:
        wide = x
        x, w = mx_quantize(x), mx_quantize(w)
        assert torch.equal(x.dequantize(torch.bfloat16), wide)
    inds = (torch.arange(tokens) % experts).int().reshape(-1, 1).to(device)
    want = m[:, None] * (k // 32) * 2.0 ** -9 * sign
    assert torch.equal(grouped_matmul(x, w, inds).view(tokens, n).float().cpu(), want)
