"""linear against its formula in 64 bits."""
import math

import pytest
import torch

from block_util import linear_exact
from op_util import HALF_STEP, assert_within
from veymoe.linear import ACTIVATIONS, linear
from veymoe.norm import MxTensor, mx_quantize

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def _make(rows, k, n, device, seed=0, mx=False, x_pad=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k + x_pad), generator=gen).bfloat16().to(device)[:, :k]
    w = (torch.randn((n, k), generator=gen) * k ** -0.5).bfloat16().to(device)
    b = (0.5 * torch.randn(n, generator=gen)).bfloat16().to(device)
    r = torch.randn((rows, n), generator=gen).to(device)
    return (mx_quantize(x), mx_quantize(w), b, r) if mx else (x, w, b, r)


def _check(x, w, bias=None, dtype=BF16, out=None, **kw):
    got = linear(x, w, bias, dtype=dtype, out=out, **kw)
    want, err = linear_exact(x, w, bias, **kw)
    assert got.dtype == dtype and got.shape == want.shape
    assert_within(got, want, err + (want.abs() + err) * (HALF_STEP[dtype] if dtype == BF16 else 2 ** -24), str(kw.keys()))
    return got


ROWS = [1, 2, 3, 5, 8, 9, 16, 17, 33, 64, 65, 130, 257, 600]


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("rows", ROWS)
def test_rows(device, rows, mx):
    for k, n in ((64, 96), (320, 33), (1024, 200), (2080, 515)):
        x, w, b, r = _make(rows, k, n, device, rows + k, mx)
        _check(x, w, dtype=FP32)
        _check(x, w, b, activation="silu", residual=r)
        if n % 2 == 0:
            _check(x, w, b, activation="swiglu")


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("k,n", [(8, 1), (32, 1), (32, 2), (40, 7), (64, 64), (96, 65), (128, 31), (160, 130), (992, 257),
                                 (1000, 64), (2560, 640), (4096, 100)])
def test_odd_sizes(device, k, n, mx):
    if mx and k % 32:
        k = k // 32 * 32 + 32
    for rows in (1, 4, 21, 140):
        x, w, b, r = _make(rows, k, n, device, k + n, mx)
        _check(x, w, b.float(), residual=r.bfloat16(), dtype=FP32)
        if n % 2 == 0:
            _check(x, w, activation="swiglu", residual=r[:, :n // 2])


@pytest.mark.parametrize("activation", list(ACTIVATIONS), ids=str)
@pytest.mark.parametrize("rows", [1, 30, 200])
def test_activations(device, rows, activation):
    """Sums up to about 60 in magnitude, over which every activation is flat, steep and curved somewhere."""
    x, w, b, r = _make(rows, 256, 128, device, rows)
    w = (w.float() * torch.linspace(0.02, 20, 128, device=device)[:, None]).bfloat16()
    n = 64 if activation == "swiglu" else 128
    for dtype in (BF16, FP32):
        for bias in (None, b, b.float()):
            _check(x, w, bias, activation=activation, dtype=dtype)
            _check(x, w, bias, activation=activation, dtype=dtype, residual=r[:, :n])
            _check(x, w, bias, activation=activation, dtype=dtype, residual=r[:, :n].bfloat16().contiguous())


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("rows,k,n", [(2048, 512, 512), (1030, 320, 1400), (2100, 1024, 700), (700, 2560, 2568)])
def test_larger_calls(device, rows, k, n, mx):
    x, w, b, r = _make(rows, k, n, device, 1, mx)
    _check(x, w, b, activation="gelu", residual=r.bfloat16())
    _check(x, w, activation="swiglu", dtype=FP32)


def test_strides(device):
    x, w, b, r = _make(20, 128, 48, device, 2, x_pad=64)
    _check(x, w, b, residual=r)
    big = torch.randn((96, 256), device=device).bfloat16()
    _check(x, big[::2, 64:192], residual=r)                      # every other row, from the middle
    _check(big[:1, :128].expand(7, 128), w)
    _check(x.reshape(4, 5, 128), w, residual=r.view(4, 5, 48))
    _check(x[0], w, residual=r[0])
    wide = torch.full((22, 80), 7.0, dtype=FP32, device=device)
    got = _check(x, w, b, dtype=FP32, out=wide[1:21, 9:57])
    assert got.data_ptr() == wide[1:21, 9:57].data_ptr()
    wide[1:21, 9:57] = 7.0
    assert (wide == 7.0).all()
    # MX operands inside wider buffers; scales off four-byte words
    q, qw = mx_quantize(torch.randn((30, 352), device=device)), mx_quantize(torch.randn((50, 352), device=device))
    cut = lambda t, lo, hi: MxTensor(t.values[:, lo:hi], t.scales[:, lo // 32:hi // 32])  # noqa: E731
    for lo, hi in ((0, 352), (32, 352), (64, 96), (96, 320), (128, 256)):
        _check(cut(q, lo, hi), cut(qw, lo, hi), dtype=FP32)


def test_in_place_over_the_residual(device):
    for rows in (1, 12, 300):
        for dtype in (BF16, FP32):
            x, w, b, r = _make(rows, 256, 200, device, 3)
            r = r.to(dtype)
            want = linear(x, w, b, activation="relu", residual=r, dtype=dtype)
            mine = r.clone()
            got = linear(x, w, b, activation="relu", residual=mine, dtype=dtype, out=mine)
            assert got is mine and torch.equal(got, want)


def test_not_numbers_stay_where_they_are(device):
    """A NaN in a row, a matrix row, a bias or a residual reaches its own outputs only; infinities come through."""
    for rows in (3, 40, 300):
        for activation in (None, "relu", "silu", "gelu", "swiglu"):
            x, w, b, r = _make(rows, 72, 80, device, 4)
            n = 40 if activation == "swiglu" else 80
            x[1, 71], w[5, 70], b[7], r[0, 9] = math.nan, math.nan, math.nan, math.inf
            got = linear(x, w, b, activation=activation, residual=r[:, :n], dtype=FP32).cpu()
            bad = torch.zeros((rows, n), dtype=torch.bool)
            bad[1], bad[:, 5], bad[:, 7] = True, True, True
            assert torch.equal(torch.isnan(got), bad)
            assert got[0, 9] == math.inf and (got[2, 9] != math.inf)


def test_sums_of_cancelling_terms(device):
    """Large terms that cancel leave the small ones, to fp32's last bits: 2^12 + 1 - 2^12, one term to a k."""
    for rows in (1, 20, 200):
        k = 128
        x = torch.zeros((rows, k), dtype=BF16, device=device)
        w = torch.ones((64, k), dtype=BF16, device=device)
        x[:, 0], x[:, 9], x[:, 70] = 4096.0, 1.0, -4096.0
        assert (linear(x, w, dtype=FP32) == 1.0).all()
        q, qw = mx_quantize(x), mx_quantize(w)
        assert (linear(q, qw, dtype=FP32) == 1.0).all()


def test_repeats_empty_and_scales(device):
    x, w, b, r = _make(333, 512, 300, device, 5)
    assert torch.equal(linear(x, w, b, residual=r), linear(x, w, b, residual=r))
    assert linear(x[:0], w).shape == (0, 300) and linear(x, w[:0]).shape == (333, 0)
    q = mx_quantize(x)
    a = linear(q, mx_quantize(w))
    assert torch.equal(a, linear(MxTensor(q.values, q.scales.view(torch.uint8)), mx_quantize(w)))
