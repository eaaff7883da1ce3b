"""grouped_matmul against the definition in 64 bits."""
import pytest
import torch

from op_util import HALF_STEP, assert_mx_within, assert_within, mx_value, product_exact
from veymoe.norm import MxTensor, mx_quantize
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu


def _ids(gen, tokens, slots, experts):
    return torch.stack([torch.randperm(experts, generator=gen)[:slots] for _ in range(tokens)]).int().reshape(tokens, slots)


def _operands(gen, x_shape, w_shape, mx, device):
    x = torch.randn(x_shape, generator=gen).bfloat16().to(device)
    w = (torch.randn(w_shape, generator=gen) * w_shape[-1] ** -0.5).bfloat16().to(device)
    return (mx_quantize(x), mx_quantize(w)) if mx else (x, w)


def _wide(t):
    return mx_value(t) if isinstance(t, MxTensor) else t.cpu().double()


def _check(x, w, inds, swiglu, quantize, shared, **kw):
    got = grouped_matmul(x, w, inds, activation="swiglu" if swiglu else None, quantize=quantize, **kw)
    rows = _wide(x)
    if shared:
        rows = rows[..., None, :].expand(*inds.shape, rows.shape[-1])
    want, err = product_exact(rows, _wide(w), inds, swiglu)
    if quantize:
        assert_mx_within(got, want, err)
    else:
        assert_within(got, want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])
    return got


# tokens, slots, experts, k, n: rows one by one (short and long k), tiles of 32 and 64 rows, with full and ragged
# last tiles, k of whole chunks or not, n off every tile size, one expert, more experts than rows
SIZES = [(1, 10, 512, 256, 64), (1, 1, 1, 32, 32), (3, 10, 64, 2048, 96), (2, 4, 9, 1056, 160),
         (8, 10, 100, 640, 320), (24, 10, 512, 256, 96), (33, 1, 7, 2048, 32), (20, 4, 64, 1088, 224),
         (90, 4, 8, 256, 64), (100, 3, 6, 160, 96), (300, 2, 9, 384, 256), (333, 4, 64, 224, 128),
         (130, 1, 1, 512, 96), (700, 4, 16, 256, 160), (515, 2, 8, 96, 32), (1200, 4, 20, 128, 64),
         (1024, 4, 128, 96, 96), (1024, 4, 129, 96, 96), (1025, 4, 40, 96, 96), (2047, 1, 128, 64, 160), (20, 4, 9, 160, 96),
         (27, 3, 9, 160, 96)]


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("kind", ["plain", "swiglu", "swiglu_mx"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", SIZES)
def test_products(device, tokens, slots, experts, k, n, kind, mx):
    gen = torch.Generator().manual_seed(tokens * 1000 + k + n)
    swiglu = kind != "plain"
    x, w = _operands(gen, (tokens, k), (experts, n * (2 if swiglu else 1), k), mx, device)
    inds = _ids(gen, tokens, slots, experts).to(device)
    _check(x, w, inds, swiglu, kind == "swiglu_mx", True)


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", [(2, 10, 40, 640, 2560), (32, 10, 60, 640, 70), (60, 4, 8, 256, 1001),
                                                      (200, 4, 6, 96, 130), (9, 1, 3, 2080, 1), (50, 2, 30, 64, 3)])
def test_a_row_per_slot_and_odd_outputs(device, tokens, slots, experts, k, n, mx):
    gen = torch.Generator().manual_seed(k + n)
    x, w = _operands(gen, (tokens, slots, k), (experts, n, k), mx, device)
    _check(x, w, _ids(gen, tokens, slots, experts).to(device), False, False, False)


@pytest.mark.parametrize("k,n", [(8, 5), (24, 64), (72, 33), (1000, 40), (1032, 100)])
@pytest.mark.parametrize("tokens", [1, 40, 300, 900])
def test_bf16_of_odd_inputs(device, tokens, k, n):
    gen = torch.Generator().manual_seed(tokens + k)
    x, w = _operands(gen, (tokens, k), (6, n, k), False, device)
    _check(x, w, _ids(gen, tokens, 2, 6).to(device), False, False, True)


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [5, 60, 400, 5000])
def test_ids_without_an_expert_and_repeated_ids(device, tokens, mx):
    """Rows of ids outside the experts are zero, whatever was in the output; an expert twice in one token counts
    twice; experts that no row names stay out.  5000 tokens sort over several blocks."""
    gen = torch.Generator().manual_seed(tokens)
    x, w = _operands(gen, (tokens, 64), (10, 64, 64), mx, device)
    inds = torch.randint(-1, 12, (tokens, 3), generator=gen, dtype=torch.int64)
    inds[inds == 4] = 5
    inds[0] = torch.tensor([2 ** 32 + 1, -2 ** 40, 7])
    inds[1:3] = 3
    inds[tokens - 1] = -1
    inds = inds.to(device)
    out = torch.full((tokens, 3, 32), float("nan"), dtype=torch.bfloat16, device=device)
    got = _check(x, w, inds, True, False, True, out=out)
    assert got is out
    none = ((inds < 0) | (inds >= 10)).cpu()
    assert (got.cpu()[none] == 0).all()
    assert torch.equal(grouped_matmul(x, w, inds, activation="swiglu"), got)
    q = _check(x, w, inds, True, True, True)
    assert (q.values.view(torch.uint8).cpu()[none] == 0).all() and (q.scales.view(torch.uint8).cpu()[none] == 0).all()


@pytest.mark.parametrize("tokens", [3, 100, 700])
def test_every_row_to_one_expert_and_none_to_any(device, tokens):
    gen = torch.Generator().manual_seed(1)
    x, w = _operands(gen, (tokens, 128), (5, 96, 128), False, device)
    _check(x, w, torch.full((tokens, 1), 4, dtype=torch.int32, device=device), False, False, True)
    got = grouped_matmul(x, w, torch.full((tokens, 2), 5, dtype=torch.int32, device=device))
    assert (got == 0).all()


def test_a_row_with_infinities_keeps_to_itself(device):
    gen = torch.Generator().manual_seed(2)
    for tokens in (4, 200):
        x, w = _operands(gen, (tokens, 72), (3, 64, 72), False, device)
        inds = (torch.arange(tokens) % 3).int().reshape(-1, 1).to(device)
        clean = grouped_matmul(x, w, inds)
        x[1, 70], x[2, 3] = float("inf"), float("nan")
        got = grouped_matmul(x, w, inds)
        keep = [i for i in range(tokens) if i not in (1, 2)]
        assert torch.equal(got[keep], clean[keep])
        assert not torch.isfinite(got[1]).any() and torch.isnan(got[2]).all()


@pytest.mark.parametrize("tokens", [3, 60, 200])
def test_mx_groups_that_are_not_numbers(device, tokens):
    """A row with a NaN group makes its own outputs NaN and no others'; so does a matrix row its own column."""
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, 160), generator=gen).to(device)
    w = torch.randn((4, 64, 160), generator=gen).to(device)
    inds = (torch.arange(tokens) % 4).int().reshape(-1, 1).to(device)
    clean = grouped_matmul(mx_quantize(x), mx_quantize(w), inds)
    x[1, 159], w[2, 5, 3] = float("inf"), float("nan")
    got = grouped_matmul(mx_quantize(x), mx_quantize(w), inds).view(tokens, 64)
    bad = torch.zeros((tokens, 64), dtype=torch.bool, device=device)
    bad[1] = True
    bad[inds[:, 0] == 2, 5] = True
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], clean.view(tokens, 64)[~bad])


@pytest.mark.parametrize("tokens", [4, 40, 400])
def test_mx_extremes_of_scale(device, tokens):
    """Scales far apart cancel in the product.  Below bf16's normal range values are rounded to multiples of 2^-133:
    off by 2^-134 at most, times the matrix value."""
    x, w = torch.full((tokens, 64), 1e-30), torch.full((2, 64, 64), 1e30)
    x[:, 32:] = 0
    x[3] = 1e-40
    x[2, 40] = 1e-37
    inds = torch.zeros((tokens, 1), dtype=torch.int32, device=device)
    xq, wq = mx_quantize(x.to(device)), mx_quantize(w.to(device))
    xv, wv = mx_value(xq).cpu().double(), mx_value(wq).cpu().double()[0]
    want = xv @ wv.T
    err = (xv != 0).double() @ wv.abs().T * 2.0 ** -134 + 64 * 2.0 ** -24 * want.abs()
    got = grouped_matmul(xq, wq, inds).cpu().view(tokens, 64).double()
    assert ((got - want).abs() <= err + (want.abs() + err) * HALF_STEP[torch.bfloat16]).all()


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [9, 130, 700])
def test_matrices_larger_than_the_cache(device, tokens, mx):
    """More than 256 MB of matrices, which stream past the caches but for those of several tiles: most rows of the
    larger calls go to one expert."""
    gen = torch.Generator().manual_seed(tokens)
    experts, k, n = (300, 1024, 512) if not mx else (300, 1024, 1024)
    w = torch.randn((8, n, k), generator=gen).bfloat16().to(device) * k ** -0.5
    w = w.repeat((experts + 7) // 8, 1, 1)[:experts]
    x = torch.randn((tokens, k), generator=gen).bfloat16().to(device)
    if mx:
        x, w = mx_quantize(x), mx_quantize(w)
    inds = _ids(gen, tokens, 2, experts)
    inds[tokens // 3:, 0] = 5
    inds[inds[:, 0] == inds[:, 1], 1] = 6
    got = grouped_matmul(x, w, inds.to(device))
    small = MxTensor(w.values[:8], w.scales[:8]) if mx else w[:8]
    want, err = product_exact(_wide(x)[:, None].expand(tokens, 2, k), _wide(small), inds % 8, False)
    assert_within(got, want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])


# 64-row tiles of more than 16384 rows, and 32-row ones of as many experts as there may be: the widest blocks, with k of
# whole chunks and not
@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("kind", ["plain", "swiglu", "swiglu_mx"])
@pytest.mark.parametrize("tokens,slots,experts,k,n", [(4300, 4, 40, 512, 2048), (8601, 2, 40, 544, 2112),
                                                      (4000, 2, 1024, 1024, 512), (4000, 2, 1024, 1056, 576)])
def test_large_calls(device, tokens, slots, experts, k, n, kind, mx):
    gen = torch.Generator().manual_seed(tokens + k)
    swiglu = kind != "plain"
    x, w = _operands(gen, (tokens, k), (8, n, k), mx, device)
    bank = (lambda t: t.repeat((experts + 7) // 8, 1, 1)[:experts])
    full = MxTensor(bank(w.values.view(torch.uint8)).view(w.values.dtype),
                    bank(w.scales.view(torch.uint8)).view(w.scales.dtype)) if mx else bank(w)
    inds = torch.randint(-1, experts, (tokens, slots), generator=gen, dtype=torch.int32)
    got = grouped_matmul(x, full, inds.to(device), activation="swiglu" if swiglu else None, quantize=kind == "swiglu_mx")
    some = torch.cat([torch.arange(40), torch.randint(0, tokens, (300,), generator=gen), torch.arange(tokens - 40, tokens)])
    ids = torch.where(inds < 0, -1, inds % 8)[some]
    want, err = product_exact(_wide(x)[some][:, None].expand(len(some), slots, k), _wide(w), ids, swiglu)
    pick = some.to(device)
    if kind == "swiglu_mx":
        got = MxTensor(got.values.view(torch.uint8)[pick].view(got.values.dtype),
                       got.scales.view(torch.uint8)[pick].view(got.scales.dtype))
        assert_mx_within(got, want, err)
    else:
        assert_within(got[pick], want, err + (want.abs() + err) * HALF_STEP[torch.bfloat16])
        assert (got[(inds < 0).to(device)] == 0).all()


def test_two_streams_at_once(device):
    gen = torch.Generator().manual_seed(77)
    x, w = _operands(gen, (600, 256), (12, 256, 256), False, device)
    inds = [_ids(gen, 600, 4, 12).to(device) for _ in range(2)]
    want = [grouped_matmul(x, w, i, activation="swiglu") for i in inds]
    streams = [torch.cuda.Stream() for _ in inds]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(grouped_matmul(x, w, inds[j], activation="swiglu"))
    torch.cuda.synchronize()
    for j in range(2):
        for y in got[j]:
            assert torch.equal(y, want[j])


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [2, 50, 400])
def test_strided_operands(device, tokens, mx):
    """Rows inside wider buffers, weights that are a slice of a larger bank, scales off a multiple of four bytes."""
    gen = torch.Generator().manual_seed(7)
    x, w = _operands(gen, (tokens, 224), (12, 80, 224), mx, device)
    inds = _ids(gen, tokens, 3, 6).to(device)
    cut = lambda t, k: (MxTensor(t.values[..., :k], t.scales[..., :k // 32]) if mx else t[..., :k])  # noqa: E731
    part = lambda t: (MxTensor(t.values[1:12:2, 8:72], t.scales[1:12:2, 8:72]) if mx else t[1:12:2, 8:72])  # noqa: E731
    _check(cut(x, 160), part(cut(w, 160)), inds, True, False, True)
    whole = lambda t: MxTensor(t.values.contiguous(), t.scales.contiguous()) if mx else t.contiguous()  # noqa: E731
    a = grouped_matmul(cut(x, 160), part(cut(w, 160)), inds)
    b = grouped_matmul(whole(cut(x, 160)), whole(part(cut(w, 160))), inds)
    assert torch.equal(a, b)


def test_one_row_for_all_tokens(device):
    """A broadcast row, and an empty call."""
    gen = torch.Generator().manual_seed(9)
    x, w = _operands(gen, (1, 64), (4, 32, 64), False, device)
    inds = _ids(gen, 70, 2, 4).to(device)
    assert torch.equal(grouped_matmul(x.expand(70, 64), w, inds), grouped_matmul(x.repeat(70, 1), w, inds))
    assert grouped_matmul(x[:0], w, inds[:0]).shape == (0, 2, 32)


def test_in_graphs_and_on_another_stream(device):
    """Two captured calls, each with its own scratch, replayed in turn and beside eager calls."""
    gen = torch.Generator().manual_seed(4)
    x, w = _operands(gen, (200, 256), (16, 128, 256), True, device)
    inds = [_ids(gen, 200, 4, 16).to(device) for _ in range(2)]
    first = grouped_matmul(x, w, inds[0], activation="swiglu", quantize=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, kept = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.stream(side):
        for g, i in zip(graphs, inds):
            with torch.cuda.graph(g, stream=side):
                kept.append(grouped_matmul(x, w, i, activation="swiglu", quantize=True))
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        for i in inds:
            i.copy_(_ids(gen, 200, 4, 16))
        graphs[n % 2].replay()
        graphs[1 - n % 2].replay()
        for k, i in zip(kept, inds):
            eager = grouped_matmul(x, w, i, activation="swiglu", quantize=True)
            torch.cuda.synchronize()
            assert torch.equal(k.values.view(torch.uint8), eager.values.view(torch.uint8)), n
            assert torch.equal(k.scales.view(torch.uint8), eager.scales.view(torch.uint8)), n
    assert first.values.shape == kept[0].values.shape


def test_refusals(device):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    w = torch.zeros((3, 32, 64), dtype=torch.bfloat16, device=device)
    inds = torch.zeros((4, 2), dtype=torch.int32, device=device)
    qx, qw = mx_quantize(x), mx_quantize(w)
    with pytest.raises(TypeError):
        grouped_matmul(x, qw, inds)
    with pytest.raises(TypeError):
        grouped_matmul(x.float(), w, inds)
    with pytest.raises(TypeError):
        grouped_matmul(x, w.half(), inds)
    with pytest.raises(TypeError):
        grouped_matmul(x, w, inds.float())
    with pytest.raises(TypeError):
        grouped_matmul(x.cpu(), w, inds)
    with pytest.raises(ValueError):
        grouped_matmul(x[:3], w, inds)
    with pytest.raises(ValueError):
        grouped_matmul(x, w, inds, activation="gelu")
    with pytest.raises(ValueError):
        grouped_matmul(x, w, inds, quantize=True)
    with pytest.raises(ValueError):
        grouped_matmul(x, w[:, :31], inds, activation="swiglu")
    with pytest.raises(ValueError):
        grouped_matmul(qx, qw, inds, activation="swiglu", quantize=True)   # 16 outputs: half a group
    with pytest.raises(ValueError):
        grouped_matmul(x, w, inds, out=torch.zeros((4, 2, 31), dtype=torch.bfloat16, device=device))
    with pytest.raises(ValueError):
        grouped_matmul(x, w.transpose(1, 2), inds)
    with pytest.raises(ValueError):
        grouped_matmul(MxTensor(qx.values, qx.scales[:, :1]), qw, inds)
    with pytest.raises(RuntimeError):
        grouped_matmul(x[:, :60].contiguous(), w[:, :, :60].contiguous(), inds)      # k not a multiple of 8
    with pytest.raises(ValueError):
        grouped_matmul(x[:, 1:57], w[:, :, :56], inds)                               # rows off 16 bytes
    with pytest.raises(ValueError):
        both = torch.zeros((8, 64), dtype=torch.bfloat16, device=device)
        grouped_matmul(both, w, inds[:, :1].repeat(2, 1), out=both.view(16, 32)[:8].view(8, 1, 32))
    with pytest.raises(ValueError):
        many = torch.zeros((1, 1), dtype=torch.int32, device=device).expand(2 ** 16 + 1, 2 ** 16)
        grouped_matmul(x[:1].expand(2 ** 16 + 1, 64), w, many)
