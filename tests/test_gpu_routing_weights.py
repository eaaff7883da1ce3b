"""select_experts' weights are rounded once, from 64 bits to their type."""
import pytest
import torch

from veymoe.routing import select_experts

pytestmark = pytest.mark.gpu


def _to_bf16(v):
    """The nearest bf16 value of a positive float in 64 bits, ties to even, in 64 bits."""
    m, e = torch.frexp(torch.tensor(v, dtype=torch.float64))
    step = 2.0 ** (max(int(e), -125) - 8)
    return float(torch.round(torch.tensor(v, dtype=torch.float64) / step)) * step


@pytest.mark.parametrize("rest", [0.0, 2.0 ** -45, -2.0 ** -45, 2.0 ** -30, -2.0 ** -30])
@pytest.mark.parametrize("at", [1.0, 2.0 ** -20, 2.0 ** 30, 2.0 ** -126, 2.0 ** 120])
def test_bf16_weights_next_to_halves(device, at, rest):
    """A sigmoid of one half times twice a factor that lies next to the middle of two bf16 values: fp32 does not tell it from
    the middle."""
    for j in range(8):
        factor = at * (1.0 + (2 * j + 1) * 2.0 ** -8 + rest)
        inds, weights = select_experts(torch.zeros((3, 64), device=device), 2, scoring="sigmoid", renormalize=False,
                                       scale=2.0 * factor, dtype=torch.bfloat16)
        assert weights.cpu().double().tolist() == [[_to_bf16(factor)] * 2] * 3, (j, factor)
        neg = select_experts(torch.zeros((3, 64), device=device), 2, scoring="sigmoid", renormalize=False, scale=-2.0 * factor,
                             dtype=torch.bfloat16)[1]
        assert torch.equal(neg, -weights)


@pytest.mark.parametrize("factor", [2.0 ** -133 * (2.5 + 2.0 ** -30), 2.0 ** -133 * (2.5 - 2.0 ** -30), 2.0 ** -134 * (1 + 2.0 ** -40),
                                    2.0 ** -134, 2.0 ** -160, 2.0 ** 128 * (1 - 2.0 ** -9 - 2.0 ** -40)])
def test_bf16_weights_at_the_ends(device, factor):
    weights = select_experts(torch.zeros((1, 8), device=device), 1, scoring="sigmoid", renormalize=False, scale=2.0 * factor,
                             dtype=torch.bfloat16)[1]
    assert float(weights) == _to_bf16(factor)


def test_bf16_weights_past_the_end(device):
    weights = select_experts(torch.zeros((1, 8), device=device), 1, scoring="sigmoid", renormalize=False,
                             scale=2.0 ** 129 * (1 - 2.0 ** -9), dtype=torch.bfloat16)[1]
    assert float(weights) == float("inf")
