"""add_adapters against the definition in 64 bits."""
import pytest
import torch

from op_util import HALF_STEP, adapters_exact, assert_within
from veymoe.adapters import add_adapters

pytestmark = pytest.mark.gpu


def _bank(gen, rows, k, n, rank, adapters, device, none=0.2):
    base, x = torch.randn((rows, n), generator=gen), torch.randn((rows, k), generator=gen)
    a = torch.randn((adapters, rank, k), generator=gen) * k ** -0.5
    b = torch.randn((adapters, n, rank), generator=gen) * rank ** -0.5
    ids = torch.randint(0, adapters, (rows,), generator=gen, dtype=torch.int32)
    ids[torch.rand(rows, generator=gen) < none] = -1
    return [t.bfloat16().to(device) for t in (base, x, a, b)] + [ids.to(device)]


def _check(base, x, a, b, ids, scales=None, **kw):
    want, err = adapters_exact(base, x, a, b, ids, scales)
    got = add_adapters(base, x, a, b, ids, scales=scales, **kw)
    assert_within(got, want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])
    return got


# rows one by one, tiles of 16 (one sort block and several), ranks of one to eight fragments and between, k and n off
# every vector size
SIZES = [(1, 256, 256, 16, 4), (1, 2560, 2560, 16, 3), (5, 1000, 300, 32, 9), (128, 64, 1030, 8, 2), (17, 77, 51, 7, 5),
         (129, 256, 256, 16, 4), (200, 640, 1280, 64, 7), (333, 1000, 77, 33, 64), (300, 75, 130, 5, 3),
         (257, 128, 64, 128, 2), (400, 64, 256, 1, 1), (5000, 64, 96, 24, 40), (600, 2048, 1024, 17, 600),
         (512, 64, 40, 12, 30), (513, 64, 40, 12, 30), (100, 256, 520, 64, 9), (101, 256, 520, 64, 9), (70, 40, 72, 96, 2),
         (2048, 64, 64, 8, 1024), (2048, 64, 72, 16, 3), (2049, 64, 64, 8, 1024), (1999, 72, 64, 40, 257), (128, 96, 64, 16, 30), (129, 96, 64, 16, 30),
         (7, 96, 64, 64, 30), (8, 96, 64, 64, 30), (4, 96, 264, 128, 3)]


@pytest.mark.parametrize("rows,k,n,rank,adapters", SIZES)
def test_adapters(device, rows, k, n, rank, adapters):
    gen = torch.Generator().manual_seed(rows + k)
    base, x, a, b, ids = _bank(gen, rows, k, n, rank, adapters, device)
    scales = (torch.rand(adapters, generator=gen) * 2 - 0.5).to(device)
    got = _check(base, x, a, b, ids, scales)
    assert torch.equal(got[ids < 0], base[ids < 0])
    _check(base, x, a, b, ids)
    again = base.clone()
    assert add_adapters(again, x, a, b, ids, scales=scales, out=again) is again
    assert torch.equal(again, got)


@pytest.mark.parametrize("rows", [6, 300])
def test_adapters_ids_strides_and_dimensions(device, rows):
    """64-bit ids far outside stay outside; rows inside wider buffers, aligned and not; leading dimensions."""
    gen = torch.Generator().manual_seed(8)
    base, x, a, b, ids = _bank(gen, rows, 128, 96, 16, 5, device, 0.0)
    wide = ids.long()
    wide[1], wide[2], wide[3] = 2 ** 32 + 1, 5, -2 ** 40
    want = _check(base, x, a, b, wide)
    assert torch.equal(want[1:4], base[1:4])
    for pad in (8, 3):
        bw, xw = torch.zeros((rows, 96 + pad)), torch.zeros((rows, 128 + pad))
        bw, xw = bw.bfloat16().to(device), xw.bfloat16().to(device)
        bw[:, :96], xw[:, :128] = base, x
        out = torch.zeros((rows, 200), dtype=torch.bfloat16, device=device)
        add_adapters(bw[:, :96], xw[:, :128], a, b, wide, out=out[:, pad:pad + 96])
        # the scalar loads sum in the same order, so the strides change no bit
        assert torch.equal(out[:, pad:pad + 96], want)
        assert (out[:, :pad] == 0).all() and (out[:, pad + 96:] == 0).all()
    got = add_adapters(base.view(2, rows // 2, 96), x.view(2, rows // 2, 128), a, b, wide.view(2, rows // 2))
    assert torch.equal(got.view(rows, 96), want)
    assert add_adapters(base[:0], x[:0], a, b, ids[:0]).shape == (0, 96)


@pytest.mark.parametrize("rows", [9, 600])
def test_adapters_of_banks_off_the_vector_units(device, rows):
    """Banks that start two bytes into a buffer take element loads; the results stay the same."""
    gen = torch.Generator().manual_seed(rows)
    base, x, a, b, ids = _bank(gen, rows, 128, 96, 16, 5, device)
    want = _check(base, x, a, b, ids)
    for which in ("a", "b", "ab"):
        banks = []
        for name, t in (("a", a), ("b", b)):
            off = torch.empty(t.numel() + 1, dtype=torch.bfloat16, device=device)[1:].view(t.shape)
            banks.append(off.copy_(t) if name in which else t)
        got = _check(base, x, *banks, ids)
        assert torch.equal(got[ids < 0], want[ids < 0])


def test_adapters_of_many_rows_and_as_many_as_may_be(device):
    gen = torch.Generator().manual_seed(16385)
    for rows, k, n, rank, adapters in ((16385, 64, 72, 16, 3), (40000, 32, 40, 8, 1024), (16384, 32, 64, 8, 1024)):
        base, x, a, b, ids = _bank(gen, rows, k, n, rank, adapters, device)
        ids[:3] = adapters - 1
        _check(base, x, a, b, ids)


def test_adapters_side_by_side_in_one_buffer(device):
    """base, x and out as column ranges of the same rows do not overlap."""
    gen = torch.Generator().manual_seed(5)
    base, x, a, b, ids = _bank(gen, 700, 64, 96, 16, 5, device)
    rows = torch.zeros((700, 96 + 64 + 96), dtype=torch.bfloat16, device=device)
    rows[:, :96], rows[:, 96:160] = base, x
    want = add_adapters(base, x, a, b, ids)
    got = add_adapters(rows[:, :96], rows[:, 96:160], a, b, ids, out=rows[:, 160:])
    assert torch.equal(got, want)
    assert torch.equal(rows[:, :96], base) and torch.equal(rows[:, 96:160], x)


@pytest.mark.parametrize("rows", [4, 200])
def test_adapters_without_any_and_with_one(device, rows):
    gen = torch.Generator().manual_seed(12)
    base, x, a, b, ids = _bank(gen, rows, 64, 64, 8, 3, device)
    assert torch.equal(add_adapters(base, x, a, b, torch.full_like(ids, -1)), base)
    _check(base, x, a, b, torch.full_like(ids, 2))
    x[1] = float("nan")
    got = add_adapters(base, x, a, b, torch.full_like(ids, 2))
    assert torch.isnan(got[1]).all() and torch.isfinite(got[2:]).all() and torch.isfinite(got[0]).all()


def test_adapters_in_a_graph(device):
    gen = torch.Generator().manual_seed(6)
    base, x, a, b, ids = _bank(gen, 300, 256, 512, 32, 6, device)
    add_adapters(base, x, a, b, ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kept = add_adapters(base, x, a, b, ids)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        ids.copy_(torch.randint(-1, 6, (300,), generator=gen, dtype=torch.int32))
        graph.replay()
        eager = add_adapters(base, x, a, b, ids)
        torch.cuda.synchronize()
        assert torch.equal(kept, eager), n


def test_adapters_refusals(device):
    gen = torch.Generator().manual_seed(1)
    base, x, a, b, ids = _bank(gen, 4, 64, 32, 8, 3, device)
    with pytest.raises(TypeError):
        add_adapters(base.float(), x, a, b, ids)
    with pytest.raises(TypeError):
        add_adapters(base, x, a.float(), b, ids)
    with pytest.raises(TypeError):
        add_adapters(base, x, a, b, ids.float())
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b.transpose(1, 2), ids)
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b[:, :16].contiguous(), ids)
    with pytest.raises(ValueError):
        add_adapters(base, x[:3], a, b, ids)
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b, ids[:3])
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b, ids, scales=torch.ones(2, device=device))
    with pytest.raises(RuntimeError):
        add_adapters(base, x, a.repeat(1, 17, 1), b.repeat(1, 1, 17), ids)    # rank 136
    with pytest.raises(ValueError):
        add_adapters(base, x[:, :32], a[:, :, :32].contiguous(), b, ids, out=x[:, :32])
    with pytest.raises(ValueError):
        both = torch.zeros((5, 32), dtype=torch.bfloat16, device=device)
        add_adapters(both[:4], x, a, b, ids, out=both[1:])
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b, ids, out=base[:1].expand(4, 32))          # one row for all results
    with pytest.raises(ValueError):
        add_adapters(base, x, a, b, ids, scales=0.5)
