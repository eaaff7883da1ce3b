"""add_adapters where the rank sums' own bits show: the rows' form and the tiled one hold them in fp32 alike."""
import pytest
import torch

from op_util import HALF_STEP, adapters_exact, assert_within
from veymoe.adapters import add_adapters

pytestmark = pytest.mark.gpu

# rows one by one, tiles that each block finds, tiles behind a sort; ranks of one to eight fragments and off eight
ROWS, RANKS = [3, 700, 2100], [8, 16, 18, 32, 40, 64, 128]


@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("rows", ROWS)
def test_rank_sums_that_cancel(device, rows, rank):
    """Rank sums 1 + 2^-9 + m 2^-20 and 1 + 2^-9 in turn, which B subtracts: every step is exact in fp32, and so is the
    difference of at most 64 m, m up to 3 (eight bits), in bf16."""
    k, n = 192, 72
    m = (torch.arange(rows) % 3 + 1).float()
    x = torch.zeros(rows, k)
    x[:, 0], x[:, 64], x[:, 130] = 1.0, 2.0 ** -9, m * 2.0 ** -20    # chunks of different waves
    a = torch.zeros(2, rank, k)
    a[:, :, 0], a[:, :, 64], a[:, 0::2, 130] = 1.0, 1.0, 1.0
    b = torch.ones(2, n, rank)
    b[:, :, 1::2] = -1.0
    b[1] = -b[1]
    ids = (torch.arange(rows) % 2).int()
    args = [t.bfloat16().to(device) for t in (torch.zeros(rows, n), x, a, b)]
    want = m * (rank // 2) * 2.0 ** -20 * torch.where(ids == 0, 1.0, -1.0)
    got = add_adapters(*args, ids.to(device))
    assert torch.equal(got.float().cpu(), want[:, None].expand(rows, n))


@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("rows", ROWS)
def test_rank_sums_that_only_fp32_holds(device, rows, rank):
    """Sums of 511.5 * 2^119, finite in fp32 and infinite in bf16."""
    k, n = 64, 64
    x, a = torch.zeros(rows, k), torch.zeros(1, rank, k)
    x[:, 0], x[:, 1] = 255 * 2.0 ** 60, 1.5 * 2.0 ** 60
    a[:, :, 0], a[:, :, 1] = 2.0 ** 60, 2.0 ** 59
    b = torch.full((1, n, rank), 2.0 ** -120)
    args = [t.bfloat16().to(device) for t in (torch.ones(rows, n), x, a, b)]
    ids = torch.zeros(rows, dtype=torch.int32, device=device)
    want, err = adapters_exact(*args, ids)
    assert torch.isfinite(want).all()
    assert_within(add_adapters(*args, ids), want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])


@pytest.mark.parametrize("few_bits", [True, False], ids=["few_bits", "all_bits"])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("rows", ROWS)
def test_infinities_in_b(device, rows, rank, few_bits):
    """A column of B with an infinity gives infinities of the rank sums' sign, there and nowhere else."""
    gen = torch.Generator().manual_seed(rows + rank)
    k, n = 128, 72
    x, a = torch.randn((rows, k), generator=gen), torch.randn((3, rank, k), generator=gen)
    if few_bits:                                    # rank sums of a few bits
        x, a = torch.zeros(rows, k), torch.zeros(3, rank, k)
        x[:, 5], a[:, :, 5] = (torch.arange(rows) % 7 - 3.5), 0.5
    b, base = torch.randn((3, n, rank), generator=gen), torch.randn((rows, n), generator=gen)
    b[0, 7, rank - 1], b[1, 70, 0], b[2, 33, rank // 2] = float("inf"), float("-inf"), float("inf")
    ids = torch.randint(-1, 3, (rows,), generator=gen, dtype=torch.int32)
    args = [t.bfloat16().to(device) for t in (base, x, a, b)]
    want, err = adapters_exact(*args, ids)
    assert torch.isinf(want).sum() == (ids >= 0).sum() and not torch.isnan(want).any()
    got = add_adapters(*args, ids.to(device))
    fine = torch.isfinite(want)
    bound = torch.where(fine, err + (want.abs() + err) * HALF_STEP[torch.bfloat16], 0.0)
    assert_within(got, want, bound)
