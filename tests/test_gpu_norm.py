"""rms_norm and mx_quantize against their definitions in 64 bits."""
import pytest
import torch

from op_util import HALF_STEP, assert_mx_within, assert_within, mx_exact, mx_value, norm_exact
from veymoe.norm import MxTensor, mx_quantize, rms_norm

pytestmark = pytest.mark.gpu


def _rows(gen, rows, width, dtype, pad=0, scale=1.0):
    wide = torch.randn((rows, width + pad), generator=gen) * scale
    return wide.to(dtype).to("cuda")[:, :width]


# one row, rows of a block, of waves; a single value, widths off the vector size, of one to 16 wave steps
SHAPES = [(1, 2560), (3, 1), (5, 33), (1, 16384), (37, 2048), (2, 512), (7, 520), (1023, 96), (1024, 96), (1030, 2560),
          (1100, 1000), (1025, 4096), (1024, 4104), (1027, 777), (1500, 3585)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_norm(device, rows, width, dtype, pad):
    gen = torch.Generator().manual_seed(rows * 31 + width + pad)
    x, r = _rows(gen, rows, width, dtype, pad), _rows(gen, rows, width, dtype, 2 * pad, 3.0)
    w = torch.randn(width, generator=gen).to(dtype).to(device)
    for residual, centered in ((r, True), (None, False)):
        y, h, err = norm_exact(x, w, residual, 1e-5, centered)
        got = rms_norm(x, w, eps=1e-5, residual=residual, one_centered=centered)
        got, s = got if residual is not None else (got, None)
        assert_within(got, y, err + (y.abs() + err) * HALF_STEP[dtype], "norm")
        if s is not None:
            assert_within(s, h, h.abs() * (HALF_STEP[dtype] + 2.0 ** -24), "sum")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,pad", [(1, 2560, 0), (3, 32, 0), (37, 2048, 8), (1024, 96, 0), (1030, 2560, 40),
                                            (1025, 544, 3), (2, 16384, 0), (1026, 4096, 0)])
def test_norm_to_mx(device, rows, width, pad, dtype):
    gen = torch.Generator().manual_seed(rows + width)
    x, r = _rows(gen, rows, width, dtype, pad), _rows(gen, rows, width, dtype, pad, 3.0)
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(device)  # a float32 gain beside either type
    y, h, err = norm_exact(x, w, r)
    got, s = rms_norm(x, w, residual=r, quantize=True)
    assert isinstance(got, MxTensor) and got.scales.shape == (rows, width // 32)
    assert_mx_within(got, y, err, "mx")
    assert_within(s, h, h.abs() * (HALF_STEP[dtype] + 2.0 ** -24), "sum")
    assert torch.equal(got.dequantize().cpu().double(), mx_value(got))


def test_norm_in_place_and_leading_dimensions(device):
    gen = torch.Generator().manual_seed(5)
    x, r = (torch.randn((3, 5, 256), generator=gen).bfloat16().to(device) for _ in range(2))
    w = torch.randn(256, generator=gen).bfloat16().to(device)
    want, h = rms_norm(x, w, residual=r)
    assert want.shape == x.shape
    xs, rs = x.clone(), r.clone()
    got, s = rms_norm(xs, w, residual=rs, out=xs, residual_out=rs)
    assert got is xs and s is rs
    assert torch.equal(got, want) and torch.equal(s, h)
    empty = rms_norm(x[:0], w)
    assert empty.shape == (0, 5, 256)


def test_norm_of_extremes(device):
    """Rows of zeros, of a single large value, of values near the ends of fp32, and rows with an infinity or a NaN,
    which stay their own rows'."""
    x = torch.zeros(6, 64)
    x[1, 3] = 3e38
    x[2] = 1e-30
    x[3, 0], x[4, 1] = float("inf"), float("nan")
    x[5] = torch.arange(64.0) - 31
    w = torch.ones(64)
    got = rms_norm(x.to(device), w.to(device), eps=1e-6).cpu()
    mx = rms_norm(x.to(device), w.to(device), eps=1e-6, quantize=True)
    assert (got[0] == 0).all() and (got[1] == 0).all()      # 3e38 squared is infinite in fp32: 3e38 / inf
    assert torch.isnan(got[3, 0]) and (got[3, 1:] == 0).all() and torch.isnan(got[4]).all()
    y, _, err = norm_exact(x[[2, 5]], w)
    assert_within(got[[2, 5]], y, err + (y.abs() + err) * HALF_STEP[torch.float32])
    v = mx_value(mx)
    assert (v[:3] != v[:3]).sum() == 0 and torch.isnan(v[3, :32]).all() and (v[3, 32:] == 0).all()
    assert torch.isnan(v[4]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_mx_quantize_is_the_definition(device, dtype):
    """Every value and scale equal: powers of two, the border at 448, ties, zeros, subnormals, infinities and NaN."""
    gen = torch.Generator().manual_seed(11)
    x = torch.randn((200, 96), generator=gen) * torch.exp2(torch.randint(-30, 30, (200, 3), generator=gen).float()
                                                          ).repeat_interleave(32, 1)
    x[0] = 0
    x[1, :32], x[1, 32:64], x[1, 64:] = 448.0, 449.0, 450.0
    x[2] = 1e-44                                    # subnormal in fp32, zero in bf16
    x[3] = 2.0 ** -126
    x[4] = (torch.arange(96) % 32).float() + 0.5     # ties
    x[5, 7], x[6, 40], x[7, 90] = float("inf"), float("-inf"), float("nan")
    x[8] = 3.3e38
    x[9, ::2] = -x[9, ::2].abs()
    x = x.to(dtype)
    got = mx_quantize(x.to(device))
    q, s = mx_exact(x.double())
    mine = torch.exp2(got.scales.view(torch.uint8).cpu().double() - 127)
    mine[got.scales.view(torch.uint8).cpu() == 255] = float("nan")
    assert torch.equal(torch.isnan(mine), torch.isnan(s)) and torch.equal(mine[~torch.isnan(s)], s[~torch.isnan(s)])
    v = got.values.cpu().float().double()
    assert torch.equal(torch.isnan(v), torch.isnan(q)) and torch.equal(v[~torch.isnan(q)], q[~torch.isnan(q)])


def test_norm_on_another_stream_and_in_a_graph(device):
    gen = torch.Generator().manual_seed(3)
    x, r = (torch.randn((64, 2560), generator=gen).bfloat16().to(device) for _ in range(2))
    w = torch.randn(2560, generator=gen).bfloat16().to(device)
    want, h = rms_norm(x, w, residual=r, quantize=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = rms_norm(x, w, residual=r, quantize=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept, kept_h = rms_norm(x, w, residual=r, quantize=True)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=gen).bfloat16())
        graph.replay()
        fresh, fresh_h = rms_norm(x, w, residual=r, quantize=True)
        torch.cuda.synchronize()
        assert torch.equal(kept.values.view(torch.uint8), fresh.values.view(torch.uint8)), n
        assert torch.equal(kept.scales.view(torch.uint8), fresh.scales.view(torch.uint8)), n
        assert torch.equal(kept_h, fresh_h), n
    assert torch.equal(other.values.view(torch.uint8), want.values.view(torch.uint8))


def test_norm_refusals(device):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    w = torch.ones(64, dtype=torch.bfloat16, device=device)
    with pytest.raises(TypeError):
        rms_norm(x.half(), w)
    with pytest.raises(TypeError):
        rms_norm(x.cpu(), w)
    with pytest.raises(ValueError):
        rms_norm(x, w[:32])
    with pytest.raises(ValueError):
        rms_norm(x, w, residual=x[:2])
    with pytest.raises(TypeError):
        rms_norm(x, w, residual=x.float())
    with pytest.raises(ValueError):
        rms_norm(x.t(), w[:4])
    with pytest.raises(ValueError):
        rms_norm(x[:, :40].contiguous(), w[:40], quantize=True)
    with pytest.raises(ValueError):
        rms_norm(x, w, residual_out=x)
    with pytest.raises(ValueError):
        rms_norm(x.view(2, 2, 64)[:, :1].expand(2, 3, 64), w)       # rows without one stride
    with pytest.raises(ValueError):
        mx_quantize(x[:, :40])
    wide = torch.zeros((1, 16416), dtype=torch.bfloat16, device=device)
    with pytest.raises(RuntimeError):
        rms_norm(wide, torch.ones(16416, dtype=torch.bfloat16, device=device))
    with pytest.raises(ValueError):
        rms_norm(x[:, :32], w[:32], out=x[:, 16:48])
    with pytest.raises(ValueError):
        rms_norm(x, w, out=x[:1].expand(4, 64))
    with pytest.raises(ValueError):
        rms_norm(x, w, residual=x.clone(), out=x, residual_out=x)
    with pytest.raises(ValueError):
        rms_norm(x[:1, :1].expand(2 ** 32 + 2, 1), w[:1])


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float32])
def test_norm_over_its_operands(device, act):
    """The normed rows over residual and h over x, and all of them as column ranges of one buffer."""
    gen = torch.Generator().manual_seed(3)
    x, r = (torch.randn((1500, 96), generator=gen).to(act).to(device) for _ in range(2))
    w = torch.rand(96, generator=gen).to(device)
    y, h = rms_norm(x, w, residual=r)
    xs, rs = x.clone(), r.clone()
    rms_norm(xs, w, residual=rs, out=rs, residual_out=xs)
    assert torch.equal(rs, y) and torch.equal(xs, h)
    buf = torch.cat([x, r, torch.zeros_like(x), torch.zeros_like(x)], 1)
    parts = buf.split(96, 1)
    rms_norm(parts[0], w, residual=parts[1], out=parts[2], residual_out=parts[3])
    for part, want in zip(parts, (x, r, y, h)):
        assert torch.equal(part, want)


def test_dequantize_of_the_least_scales(device):
    x = torch.zeros((2, 64), device=device)
    x[0, :32], x[0, 32:], x[1, :32], x[1, 32:] = 2.0 ** -127, 3.0 * 2.0 ** -128, 2.0 ** 127, 2.0 ** -110
    assert torch.equal(mx_quantize(x).dequantize(), x)
    assert torch.equal(mx_quantize(x).dequantize(torch.bfloat16), x.bfloat16())


@pytest.mark.parametrize("rows", [3, 2000])
def test_norm_to_mx_with_a_gain_of_one_and_weight(device, rows):
    gen = torch.Generator().manual_seed(rows)
    x, w = torch.randn((rows, 96), generator=gen).bfloat16().to(device), (torch.rand(96, generator=gen) - 0.5).to(device)
    want, _, err = norm_exact(x, w, one_centered=False)
    assert_mx_within(rms_norm(x, w, one_centered=False, quantize=True), want, err)
