"""Rows, matrices and outputs whose offsets pass 32 bits, in elements and bytes: the same bits as side by side."""
import pytest
import torch

from veymoe.adapters import add_adapters
from veymoe.norm import MxTensor, mx_quantize, rms_norm
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu

FAR = (1 << 31) + 64        # elements between rows: the third lies past 2^32 of them


@pytest.fixture(scope="module")
def field(device):
    """Ten GiB, not initialised."""
    t = torch.empty(5 << 30, dtype=torch.bfloat16, device=device)
    yield t
    del t
    torch.cuda.empty_cache()


def _far(field, t, at=0, stride=FAR):
    """t's rows (its outer dimension) `stride` elements apart in the field, from element `at` on."""
    inner = t[0].stride() if t.dim() > 1 else ()
    base = field if t.dtype == field.dtype else field.view(t.dtype)
    return base.as_strided(t.shape, (stride, *inner), at).copy_(t)


def test_norm_of_far_rows(field, device):
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn((3, 96), generator=gen).bfloat16().to(device) for _ in range(2))
    w = torch.rand(96, generator=gen).to(device)
    want, h = rms_norm(x, w, residual=r)
    q, _ = rms_norm(x, w, residual=r, quantize=True)
    fx, fr = _far(field, x), _far(field, r, 96)
    out, total = _far(field, torch.zeros_like(x), 192), _far(field, torch.zeros_like(x), 288)
    rms_norm(fx, w, residual=fr, out=out, residual_out=total)
    assert torch.equal(out, want) and torch.equal(total, h) and torch.equal(fx, x) and torch.equal(fr, r)
    got, _ = rms_norm(fx, w, residual=fr, quantize=True)
    assert torch.equal(got.values.view(torch.uint8), q.values.view(torch.uint8))
    assert torch.equal(mx_quantize(fx).values.view(torch.uint8), mx_quantize(x).values.view(torch.uint8))


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("slots", [1, 60, 2000])
def test_products_of_far_rows_and_matrices(field, device, slots, mx):
    """Far token rows, far experts, and one expert's far rows; rows one by one, tiles, and tiles behind a sort."""
    gen = torch.Generator().manual_seed(slots)
    x, w = torch.randn((3, 64), generator=gen).bfloat16().to(device), torch.randn((3, 3, 64), generator=gen).bfloat16().to(device)
    inds = torch.randint(0, 3, (3, slots), generator=gen, dtype=torch.int32).to(device)
    inds[2] = 2
    none = torch.zeros_like(inds)
    if not mx:
        want, one = grouped_matmul(x, w, inds), grouped_matmul(x, w[:1], none)
        fx, fw = _far(field, x), _far(field, w, 128)
        assert torch.equal(grouped_matmul(fx, fw, inds), want)
        rows = _far(field, w[0], 1024)
        assert torch.equal(grouped_matmul(fx, rows[None], none), one)
        return
    x, w = mx_quantize(x), mx_quantize(w)
    want = grouped_matmul(x, w, inds)
    byte = lambda t, at: _far(field, t.view(torch.uint8), at, 2 * FAR).view(t.dtype)  # noqa: E731
    fx = MxTensor(byte(x.values, 0), byte(x.scales, 64))
    fw = MxTensor(byte(w.values, 128), byte(w.scales, 1024))
    assert torch.equal(grouped_matmul(fx, fw, inds), want)


@pytest.mark.parametrize("rows", [3, 800])
def test_adapters_of_large_banks(field, device, rows):
    """Banks of 2.2 G values, whose last adapter lies past 2^32 bytes; and far rows of base and out."""
    gen = torch.Generator().manual_seed(rows)
    k, n, rank, count = 17000, 16992, 128, 1024
    a, b = field[:count * rank * k].view(count, rank, k), field[count * rank * k:][:count * n * rank].view(count, n, rank)
    small = [torch.randn(shape, generator=gen).bfloat16().to(device) * 0.05 for shape in ((2, rank, k), (2, n, rank))]
    for bank, part in zip((a, b), small):
        bank[0], bank[count - 1] = part[0], part[1]
    x, base = torch.randn((rows, k), generator=gen).bfloat16().to(device), torch.randn((rows, n), generator=gen).bfloat16().to(device)
    ids = torch.randint(-1, 2, (rows,), generator=gen, dtype=torch.int32)
    ids[:3] = torch.tensor([0, 1, -1])
    want = add_adapters(base, x, *small, ids.to(device))
    assert torch.equal(add_adapters(base, x, a, b, torch.where(ids == 1, count - 1, ids).to(device)), want)


def test_adapters_of_far_rows(field, device):
    gen = torch.Generator().manual_seed(2)
    base, x = torch.randn((3, 96), generator=gen).bfloat16().to(device), torch.randn((3, 64), generator=gen).bfloat16().to(device)
    a, b = torch.randn((2, 8, 64), generator=gen).bfloat16().to(device), torch.randn((2, 96, 8), generator=gen).bfloat16().to(device)
    ids = torch.tensor([0, -1, 1], dtype=torch.int32, device=device)
    want = add_adapters(base, x, a, b, ids)
    fb, fx, out = _far(field, base), _far(field, x, 96), _far(field, torch.zeros_like(base), 192)
    assert torch.equal(add_adapters(fb, fx, a, b, ids, out=out), want)
    assert out is not want and torch.equal(out, want)
