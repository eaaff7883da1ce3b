"""select_experts against its definition in 64 bits: ids equal, weights within their last rounding."""
import math

import pytest
import torch

from block_util import INF, select_exact
from op_util import HALF_STEP
from veymoe.routing import select_experts

pytestmark = pytest.mark.gpu


def _check(logits, top_k, dtype=torch.float32, **kw):
    inds, weights = select_experts(logits, top_k, dtype=dtype, **kw)
    want, w = select_exact(logits, top_k, **kw)
    assert inds.dtype == torch.int32 and weights.dtype == dtype and inds.shape == weights.shape == want.shape
    assert torch.equal(inds.cpu(), want), (inds.cpu()[(inds.cpu() != want).reshape(-1, top_k).any(-1).reshape(inds.shape[:-1])][:2])
    got = weights.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(w))
    # one rounding of a 64-bit value (its own error is 2^-50), subnormals of fp32 included; bf16 weights come by way of fp32
    bound = w.abs() * (HALF_STEP[dtype] + 2 ** -23 * (dtype != torch.float32)) * (1 + 2 ** -20) + 2 ** -149
    assert (torch.isnan(w) | ((got - w).abs() <= bound)).all(), float(((got - w).abs() / bound).nan_to_num().max())


def _logits(rows, experts, device, seed=0, dtype=torch.float32, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, experts), generator=gen) * spread).to(dtype).to(device)


def _bias(experts, device, seed=1):
    return (torch.randn(experts, generator=torch.Generator().manual_seed(seed)) * 0.05).to(device)


SIZES = [(1, 1, 1, 1), (2, 1, 1, 2), (7, 1, 1, 3), (64, 1, 1, 64), (65, 1, 1, 8), (130, 1, 1, 6), (60, 3, 2, 4), (256, 8, 4, 8),
         (160, 16, 3, 6), (512, 1, 1, 10), (512, 8, 2, 33), (1000, 5, 2, 16), (1024, 1, 1, 40), (1024, 64, 9, 64), (640, 5, 1, 16),
         (63, 21, 4, 5), (1023, 33, 20, 12), (8, 8, 8, 8)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("experts,groups,top_groups,top_k", SIZES)
def test_sizes(device, experts, groups, top_groups, top_k, biased, scoring):
    bias = _bias(experts, device) if biased else None
    for rows, group_top, renormalize, dtype in ((1, 1, True, torch.float32), (37, 2, True, torch.bfloat16),
                                               (6, 2, False, torch.float32), (5, 1, False, torch.bfloat16)):
        _check(_logits(rows, experts, device, rows, dtype), top_k, scoring=scoring, bias=bias, groups=groups,
               top_groups=top_groups, group_top=group_top, renormalize=renormalize, scale=2.5 if rows == 37 else 1.0)


@pytest.mark.parametrize("kw", [{}, {"scoring": "sigmoid"}, {"scoring": "sigmoid", "groups": 8, "top_groups": 3, "group_top": 2},
                                {"groups": 8, "top_groups": 3}], ids=str)
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
def test_rows_that_are_closed_equal_or_not_numbers(device, kw, biased):
    l = _logits(24, 64, device, 5)
    l[0] = -INF                                  # nothing open
    l[1, 1:] = -INF                              # one open
    l[2, :60] = -INF                             # four
    l[3] = 0.25                                  # all equal
    l[4] = -0.0
    l[4, ::2] = 0.0                              # both zeros are one
    l[5, 17] = math.nan
    l[6] = math.nan
    l[7, 40] = INF
    l[8, 3:5] = INF
    l[9] = torch.finfo(torch.float32).min        # a mask of the type's lowest value: open, equal
    l[10, 5:] = torch.finfo(torch.float32).min
    l[11] = -200.0 - torch.arange(64.0)          # scores that fp32 cannot hold
    l[12] = 100.0 + torch.arange(64.0)           # sigmoids of one
    l[13, :32] = -INF
    l[14, :] = torch.tensor([1.0, 2.0]).repeat(32)
    l[15] = -800.0 - torch.arange(64.0)          # sigmoids that 64 bits cannot hold
    l[16, 1:] = -1e30
    l[17, 8:] = -INF
    l[17, 5] = math.nan
    l[18] = 1e38
    bias = None
    if biased:
        bias = _bias(64, device, 9)
        bias[11] = -INF
        bias[12] = 1e6
        bias[20:24] = bias[19]                   # experts of one bias tie where their logits do
    for renormalize in (True, False):
        _check(l, 8, bias=bias, renormalize=renormalize, **kw)
        _check(l, 1, bias=bias, renormalize=renormalize, **kw)


def test_a_bias_that_is_not_a_number_goes_first(device):
    bias = _bias(64, device)
    bias[33], bias[7] = math.nan, INF
    _check(_logits(9, 64, device), 4, scoring="sigmoid", bias=bias)
    _check(_logits(9, 64, device), 4, scoring="sigmoid", bias=bias, groups=4, top_groups=2, group_top=2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_choices_closer_than_fp32(device, scoring):
    """Biases that undo the scores up to 2^-40 of them: only 64 bits see the order."""
    gen = torch.Generator().manual_seed(3)
    l = torch.randn((1, 96), generator=gen).repeat(40, 1)
    score = torch.softmax(l.double(), -1) if scoring == "softmax" else torch.sigmoid(l.double())
    bias = (0.5 - score[0]).float()              # choices 0.5 +- 2^-26
    _check(l.to(device), 12, scoring=scoring, bias=bias.to(device))
    _check(l.to(device), 12, scoring=scoring, bias=bias.to(device), groups=8, top_groups=4, group_top=2)


def test_strides_shapes_and_types(device):
    wide = _logits(30, 300, device, 2)
    _check(wide[:, 3:259], 8, groups=8, top_groups=4, group_top=2, scoring="sigmoid", bias=_bias(256, device))
    _check(wide[:, :257], 10)
    _check(wide.bfloat16()[::2, 1:130], 5, dtype=torch.bfloat16)
    _check(wide[:, :100].reshape(5, 6, 100), 7)
    _check(wide[0, :100], 7)
    _check(wide[:1, :100].expand(9, 100), 7)
    _check(wide[:, :100], 7, bias=_bias(100, device).bfloat16(), scoring="sigmoid")
    for rows in ((0, 16), (3, 0, 16)):
        inds, weights = select_experts(torch.empty(rows, device=device), 4)
        assert inds.shape == weights.shape == (*rows[:-1], 4)


def test_many_rows_and_repeats(device):
    l = _logits(4100, 256, device, 8, torch.bfloat16)
    kw = dict(scoring="sigmoid", bias=_bias(256, device), groups=8, top_groups=4, group_top=2)
    _check(l[:700], 8, **kw)
    whole, again = select_experts(l, 8, **kw), select_experts(l, 8, **kw)
    part = select_experts(l[1000:1700], 8, **kw)
    for a, b, c in zip(whole, again, part):
        assert torch.equal(a, b) and torch.equal(a[1000:1700], c)
