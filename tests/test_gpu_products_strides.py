"""grouped_matmul over single rows and matrices of any stride."""
import pytest
import torch

from veymoe.norm import MxTensor, mx_quantize
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("slots", [1, 100])
def test_strides_that_lead_to_no_row(device, slots, mx):
    """One token, one expert or one matrix row: its stride need not be whole 16-byte units."""
    gen = torch.Generator().manual_seed(slots)
    x = torch.randn((1, 64), generator=gen).bfloat16().to(device)
    w = torch.randn((3, 32, 64), generator=gen).bfloat16().to(device)
    make = mx_quantize if mx else (lambda t: t)

    def spread(t, *strides):
        """The same values at other strides."""
        if isinstance(t, MxTensor):
            return MxTensor(*(spread(part.view(torch.uint8), *strides).view(part.dtype) for part in t))
        out = torch.empty_strided(t.shape, (*strides, 1), dtype=t.dtype, device=t.device)
        return out.copy_(t)

    inds = (torch.arange(slots) % 3).int().reshape(1, -1).to(device)
    want = grouped_matmul(make(x), make(w), inds)
    assert torch.equal(grouped_matmul(spread(make(x), 68), make(w), inds), want)
    none = torch.zeros_like(inds)
    want = grouped_matmul(make(x), make(w[:1]), none)
    assert torch.equal(grouped_matmul(make(x), spread(make(w[:1]), 2053, 64), none), want)
    want = grouped_matmul(make(x), make(w[:, :1].contiguous()), inds)
    assert torch.equal(grouped_matmul(make(x), spread(make(w[:, :1].contiguous()), 64, 67), inds), want)
