"""Every form of linear, the large tiles among them, against 64 bits: every epilogue, residuals and outputs of either type, rows
and outputs that end inside a tile, inputs that end inside a step with NaN behind them."""
import math

import pytest
import torch

from block_util import linear_exact
from linear_forms import FORMS
from op_util import HALF_STEP, assert_within
from veymoe.linear import ACTIVATIONS, linear
from veymoe.norm import MxTensor, mx_quantize

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
IDS = [f"{'mx' if f[2] else 'bf16'}-{f[0]}-{f[3]}x{f[4]}x{f[5]}" for f in FORMS]


def _wide(t, pad, fill):
    """t's rows in a wider buffer whose other bytes are `fill`."""
    big = torch.full((t.shape[0], (t.shape[1] + pad) * t.element_size()), fill, dtype=torch.uint8, device=t.device).view(t.dtype)
    big[:, :t.shape[1]] = t
    return big[:, :t.shape[1]]


def _operand(t, mx):
    if not mx:
        return _wide(t, 64, 0xff)                       # bf16 NaN
    q = mx_quantize(t)
    scales = _wide(q.scales.view(torch.uint8), 4, 0xff)
    return MxTensor(_wide(q.values.view(torch.uint8), 64, 0x7f).view(torch.float8_e4m3fn), scales)


def _rows_of(t, at):
    return MxTensor(t.values.view(torch.uint8)[at].view(torch.float8_e4m3fn), t.scales[at]) if isinstance(t, MxTensor) else t[at]


def _make(form, device, spread=True):
    _, _, mx, rows, k, matrix = form
    gen = torch.Generator(device=device).manual_seed(rows + k + matrix)
    x = torch.randn((rows, k), generator=gen, device=device).bfloat16()
    w = torch.randn((matrix, k), generator=gen, device=device) * k ** -0.5
    if spread:                                          # sums up to about 20, over which every activation bends
        w *= torch.linspace(0.05, 5, 13, device=device)[torch.arange(matrix, device=device) % 13][:, None]
    return x, w.bfloat16(), gen


@pytest.mark.parametrize("activation", list(ACTIVATIONS), ids=str)
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_values(device, form, activation):
    """The first and the last rows, which end inside a tile, and some between, by all outputs; nothing but the outputs is
    written, and all of them are numbers."""
    _, _, mx, rows, k, matrix = form
    x, w, gen = _make(form, device)
    n = matrix // 2 if activation == "swiglu" else matrix
    x, w = _operand(x, mx), _operand(w, mx)
    b = torch.randn(matrix, generator=gen, device=device)
    r = torch.randn((rows, n), generator=gen, device=device)
    at = torch.arange(rows)
    if rows > 120:
        between = torch.randint(rows, (40,), generator=torch.Generator().manual_seed(rows))
        at = torch.cat([at[:40], between, at[-40:]])
    some = _rows_of(x, at.to(device))
    for bias, residual, dtype in ((b, None, FP32), (None, r.bfloat16(), BF16), (b.bfloat16(), r, BF16), (None, r, FP32),
                                  (b, r.bfloat16(), FP32)):
        big = torch.full((rows + 2, n + 16), math.nan, dtype=dtype, device=device)
        out = big[1:-1, 8:-8]
        linear(x, w, bias, activation=activation, residual=residual, dtype=dtype, out=out)
        want, err = linear_exact(some, w, bias, activation=activation,
                                 residual=None if residual is None else residual[at.to(device)])
        assert_within(out[at.to(device)], want, err + (want.abs() + err) * HALF_STEP[dtype], str((bias is None, dtype)))
        assert torch.isfinite(out).all()
        out.fill_(math.nan)
        assert torch.isnan(big).all()


@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_rows_over_their_residual(device, form):
    _, _, mx, rows, k, matrix = form
    x, w, gen = _make(form, device)
    x, w = _operand(x, mx), _operand(w, mx)
    for activation in ("silu", "swiglu"):
        n = matrix // 2 if activation == "swiglu" else matrix
        for dtype in (BF16, FP32):
            r = torch.randn((rows, n), generator=gen, device=device).to(dtype)
            want = linear(x, w, activation=activation, residual=r, dtype=dtype)
            got = linear(x, w, activation=activation, residual=r, dtype=dtype, out=r)
            assert got is r and torch.equal(got, want) and torch.isfinite(got).all()


@pytest.mark.parametrize("activation", list(ACTIVATIONS), ids=str)
@pytest.mark.parametrize("form", FORMS, ids=IDS)
def test_not_numbers_stay_where_they_are(device, form, activation):
    """NaN in a row's last input, a matrix row's, a bias or a residual reaches its own outputs only, at the tiles' ends too."""
    _, _, mx, rows, k, matrix = form
    x, w, gen = _make(form, device, spread=False)
    n = matrix // 2 if activation == "swiglu" else matrix
    b, r = torch.zeros(matrix, device=device), torch.zeros((rows, n), device=device)
    bad = torch.zeros((rows, n), dtype=torch.bool, device=device)
    for row in {rows - 1, rows // 2}:
        x[row, k - 1] = math.nan
        bad[row] = True
    for col in {n - 1, n // 3}:
        w[col, k - 1] = math.nan
        bad[:, col] = True
    b[n // 4], r[0, n // 5], r[rows // 3, n - 2] = math.nan, math.nan, math.nan
    bad[:, n // 4], bad[0, n // 5], bad[rows // 3, n - 2] = True, True, True
    if activation == "swiglu":                          # ups
        w[n + n // 6, 0], b[n + n // 7] = math.nan, math.nan
        bad[:, n // 6], bad[:, n // 7] = True, True
    got = linear(_operand(x, mx), _operand(w, mx), b, activation=activation, residual=r, dtype=FP32)
    assert torch.equal(torch.isnan(got), bad)
    assert torch.isfinite(got[~bad]).all()


@pytest.mark.parametrize("rows,k,n,activation", [(8192, 40, 2570, None), (7937, 1000, 2559, "silu"), (8191, 72, 1285, "swiglu"),
                                                 (6001, 2080, 2051, None)])
def test_large_tiles_of_ragged_sizes_are_numbers(device, rows, k, n, activation):
    """Every output is a number, which a comparison alone does not show: a difference from NaN is above no bound."""
    gen = torch.Generator(device=device).manual_seed(rows)
    make = lambda *shape: torch.randn(shape, generator=gen, device=device).bfloat16()  # noqa: E731
    x, w = _wide(make(rows, k), 64, 0xff), _wide(make(n * (2 if activation == "swiglu" else 1), k), 64, 0xff)
    for dtype in (BF16, FP32):
        for residual in (None, make(rows, n), make(rows, n).float()):
            assert torch.isfinite(linear(x, w, activation=activation, residual=residual, dtype=dtype)).all()
