"""block_norm against its formula in 64 bits."""
import math

import pytest
import torch

from block_util import block_exact
from op_util import HALF_STEP, assert_within, mx_exact, mx_value
from veymoe.norm import block_norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _make(rows, width, device, seed=0, dtype=BF16, residual=BF16, pad=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, width + pad), generator=gen).to(dtype).to(device)[:, :width]
    r = (2 * torch.randn((rows, width + pad), generator=gen)).to(residual).to(device)[:, :width]
    w, p = (1 + 0.2 * torch.randn((2, width), generator=gen)).to(dtype).to(device)
    g = {"row": (rows, 1), "channel": (width,), "value": (rows, width)}
    g = {k: torch.randn(s, generator=gen).to(dtype).to(device) for k, s in g.items()}
    return x, r, w, p, g


def _check(x, residual, weight=None, quantize=False, **kw):
    got = block_norm(x, residual, weight, quantize=quantize, **kw)
    y, h, y_err, h_err = block_exact(x, residual, weight, **kw)
    got_h = got if weight is None else got[1]
    assert got_h.dtype == residual.dtype
    if quantize:
        # 64 bits to e4m3: the definition's values themselves
        values, scales = mx_exact(y)
        mine = mx_value(got[0])
        assert torch.equal(mine.nan_to_num(7e9), (values * scales.repeat_interleave(32, -1)).nan_to_num(7e9))
        # the float that is rounded once more, and where terms cancel the 64-bit roundings of either side, a few 2^-53 of
        # the terms each, of which h_err holds at least 2^-24 (0.7 * -4.5703125 + 3.1992... leaves 1e-16 or 0)
        h_err = h.abs() * 2 ** -24 + h_err * 2 ** -27
    elif weight is not None:
        assert got[0].dtype == x.dtype
        assert_within(got[0], y, y_err + (y.abs() + y_err) * (HALF_STEP[x.dtype] if x.dtype == BF16 else 0), "y")
    assert_within(got_h, h, h_err + (h.abs() + h_err) * (HALF_STEP[residual.dtype] if residual.dtype == BF16 else 0) + 2e-45, "h")


@pytest.mark.parametrize("width", [1, 7, 32, 64, 96, 511, 512, 1000, 1024, 2560, 2561, 4096, 5000, 8192, 16384])
@pytest.mark.parametrize("rows", [1, 5, 1030])
def test_widths(device, rows, width):
    if rows > 5 and width > 5000:
        rows = 1024
    x, r, w, p, g = _make(rows, width, device, width)
    _check(x, r, w, post_weight=p)
    if width % 32 == 0:
        _check(x, r, w, post_weight=p, gate=g["row"], quantize=True, scale=0.22)


@pytest.mark.parametrize("kind", ["none", "row", "channel", "value"])
@pytest.mark.parametrize("sigmoid", [False, True], ids=["raw", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("residual", [BF16, FP32], ids=["rbf16", "rfp32"])
def test_gates_types_and_scales(device, kind, sigmoid, dtype, residual):
    for rows, width, pad in ((3, 320, 0), (1100, 96, 8), (9, 333, 3)):
        x, r, w, p, g = _make(rows, width, device, rows, dtype, residual, pad)
        kw = dict(gate=g.get(kind), sigmoid_gate=sigmoid)
        _check(x, r, w, post_weight=p, **kw)
        _check(x, r, w - 1, post_weight=p - 1, one_centered=False, scale=0.22, residual_scale=1.41, eps=1e-3, **kw)
        _check(x, r, w, **kw)
        _check(x, r, post_weight=p, scale=-0.5, **kw)
        _check(x, r, **kw)
        if width % 32 == 0:
            _check(x, r, w, post_weight=p, quantize=True, **kw)
            _check(x, r, w - 1, one_centered=False, quantize=True, residual_scale=0.7, **kw)


def test_weights_and_gate_of_another_type(device):
    x, r, w, p, g = _make(4, 256, device, 3)
    for q in (False, True):
        _check(x, r, w.float(), post_weight=p, gate=g["channel"].float(), quantize=q)
        _check(x, r, w, post_weight=p.float(), gate=g["value"].float(), quantize=q)


def test_rows_in_place(device):
    for rows, width in ((5, 512), (1500, 2560), (7, 333), (3, 9000)):
        x, r, w, p, g = _make(rows, width, device, 7)
        want = block_norm(x, r, w, post_weight=p, gate=g["value"])
        for out, res_out in ((0, 1), (1, 0), (0, None), (None, 1)):
            both = [x.clone(), r.clone()]
            got = block_norm(both[0], both[1], w, post_weight=p, gate=g["value"], out=None if out is None else both[out],
                             residual_out=None if res_out is None else both[res_out])
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            assert out is None or got[0] is both[out]
        mine = r.clone()
        y, h = block_norm(x, mine, w, post_weight=p, gate=g["value"], residual_out=mine)
        assert torch.equal(h, want[1]) and h is mine and torch.equal(y, want[0])


def test_rows_behind_a_view_stay(device):
    """Outputs inside wider buffers leave everything around them."""
    x, r, w, p, _ = _make(6, 200, device, 1)
    a, b = torch.full((8, 256), 9.0, dtype=BF16, device=device), torch.full((8, 256), 9.0, dtype=BF16, device=device)
    y, h = block_norm(x, r, w, post_weight=p, out=a[1:7, 8:208], residual_out=b[1:7, 16:216])
    want = block_norm(x, r, w, post_weight=p)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    for buf, lo in ((a, 8), (b, 16)):
        buf[1:7, lo:lo + 200] = 9.0
        assert (buf == 9.0).all()


def test_values_that_are_large_small_or_no_numbers(device):
    x, r, w, p, g = _make(6, 128, device, 2, FP32, FP32)
    x[0], r[0] = 1e30 * x[0], 1e30 * r[0]
    x[1], r[1] = 0.0, 0.0
    x[2], r[2] = 1e-30 * x[2], 1e-30 * r[2]
    _check(x, r, w, post_weight=p)
    _check(x, r, w, post_weight=p, quantize=True)
    _check(x, r, w)
    x[3, 5], r[4, 9], x[5, 40] = math.nan, math.nan, math.inf
    for kw in ({}, {"quantize": True}):
        got = block_norm(x, r, w, post_weight=p, **kw)
        y, h, _, _ = block_exact(x, r, w, post_weight=p)
        assert torch.equal(torch.isnan(got[1].cpu()), torch.isnan(h))
        if kw:
            assert torch.equal(torch.isnan(mx_value(got[0])), torch.isnan(mx_exact(y)[0]))
        else:
            assert torch.equal(torch.isnan(got[0].cpu()), torch.isnan(y))
    # a gate that is no number behind a row's end reaches nothing: widths off the threads' steps
    x, r, w, p, _ = _make(3, 72, device, 4)
    gate = torch.full((3, 72), math.inf, dtype=BF16, device=device)
    gate[:, :71] = 1.0
    got = block_norm(x[:, :71], r[:, :71], w[:71].clone(), gate=gate[:, :71])
    assert torch.isfinite(got[0].float()).all()


def test_shapes_and_empty_rows(device):
    x, r, w, p, g = _make(12, 64, device, 6)
    flat = block_norm(x, r, w, post_weight=p, gate=g["row"])
    deep = block_norm(x.view(3, 4, 64), r.view(3, 4, 64), w, post_weight=p, gate=g["row"].view(3, 4, 1))
    assert deep[0].shape == (3, 4, 64) and torch.equal(deep[0].view(12, 64), flat[0]) and torch.equal(deep[1].view(12, 64), flat[1])
    one = block_norm(x[0], r[0], w, post_weight=p, gate=g["row"][0])
    assert torch.equal(one[0], flat[0][0]) and torch.equal(one[1], flat[1][0])
    shared = block_norm(x, r[:1].expand(12, 64), w)
    assert torch.equal(shared[0], block_norm(x, r[:1].repeat(12, 1), w)[0])
    y, h = block_norm(x[:0], r[:0], w)
    assert y.shape == h.shape == (0, 64)
