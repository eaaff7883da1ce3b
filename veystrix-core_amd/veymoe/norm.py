"""Root-mean-square norm with the residual's addition in front of it, and rows in MX.

MX rows (:class:`MxTensor`) hold e4m3 values with one power-of-two scale (e8m0) per group of 32 along the row: the
least 2^e, e >= -127, that keeps the group's largest magnitude within e4m3's 448, so that no value saturates.  A group
that holds an infinity or a NaN is NaN.  ``grouped_matmul`` multiplies them on the matrix cores, scales included.

The norm is the reference's hc_norm arithmetic (patch_rmsnorm.py:108-135) in fp32, rounded where a value is stored; fp32
and MX rows take the row's factor from 64 bits, and MX rows' products keep what fp32 would drop, so that e4m3's is the one
rounding behind the fp32 sum x + residual.  Squares are fp32: a row whose squares pass its range (values of 2^57 and
above) may come out as zeros.  The reference has no 8-bit output.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .device import ACT_DTYPES, device_call, require_32_bits, row_span

MX_GROUP = _lib.VM_MX_GROUP
_SCALE_DTYPES = (torch.float8_e8m0fnu, torch.uint8)


class MxTensor(NamedTuple):
    """``values`` [.., width] float8_e4m3fn and ``scales`` [.., width / 32] float8_e8m0fnu (or its bytes, uint8)."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype=torch.float32) -> torch.Tensor:
        """The values the rows stand for (exact in bfloat16 and float32, within their ranges)."""
        groups = self.values.float().unflatten(-1, (-1, MX_GROUP))
        scale = torch.ldexp(torch.ones((), device=groups.device), self.scales.view(torch.uint8).to(torch.int32) - 127)
        scale = torch.where(self.scales.view(torch.uint8) == 255, float("nan"), scale)
        return (groups * scale[..., None]).flatten(-2).to(dtype)


def mx_empty(shape, device) -> MxTensor:
    """An uninitialised MxTensor of ``shape``."""
    return MxTensor(torch.empty(shape, dtype=torch.float8_e4m3fn, device=device),
                    torch.empty((*shape[:-1], shape[-1] // MX_GROUP), dtype=torch.float8_e8m0fnu, device=device))


def require_mx(name: str, t) -> MxTensor:
    if not isinstance(t, MxTensor) or not all(isinstance(part, torch.Tensor) for part in t):
        raise TypeError(f"{name} must be an MxTensor of two tensors")
    if t.values.dtype != torch.float8_e4m3fn or t.scales.dtype not in _SCALE_DTYPES:
        raise TypeError(f"{name} must hold float8_e4m3fn values and float8_e8m0fnu (or uint8) scales")
    if t.values.shape[-1] % MX_GROUP or t.scales.shape != (*t.values.shape[:-1], t.values.shape[-1] // MX_GROUP):
        raise ValueError(f"{name} needs one scale per {MX_GROUP} values of a row")
    return t


def _act_dtype(name, t) -> int:
    try:
        return ACT_DTYPES[t.dtype]
    except (AttributeError, KeyError):
        raise TypeError(f"{name} must be a bfloat16 or float32 tensor") from None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor = None,
             one_centered: bool = True, quantize: bool = False, out: torch.Tensor = None,
             residual_out: torch.Tensor = None):
    """``h / sqrt(mean(h^2) + eps) * gain`` over the last dimension, h = x + residual, gain = weight (``one_centered``)
    or 1 + weight.

    x [.., width] bfloat16 or float32 with equally spaced rows, width up to 16384; residual of x's shape and type;
    weight [width] in either type.  Returns the normed rows in x's type, or as an :class:`MxTensor` with ``quantize``
    (width a multiple of 32).  With a residual it returns ``(normed, h)``, h rounded to x's type; the norm itself reads
    the unrounded sum.  ``out`` and ``residual_out`` may each be x or residual, and overlap nothing otherwise.
    """
    act = _act_dtype("x", x)
    dtype, shape, index = x.dtype, x.shape, x.get_device()
    x_at, x_stride = row_span("x", x, dtype, index)
    width, count = shape[-1], x.numel()
    if count:
        require_32_bits(count // width, width)
    weight_act = _act_dtype("weight", weight)
    if weight.shape != (width,) or not weight.is_contiguous():
        raise ValueError(f"weight must be contiguous of shape ({width},)")
    w_at, _ = row_span("weight", weight, weight.dtype, index)
    r_at = r_stride = s_at = s_stride = y_at = y_stride = values_at = scales_at = 0
    if residual is not None:
        r_at, r_stride = row_span("residual", residual, dtype, index)
        if residual_out is None:
            residual_out = torch.empty_like(x)
        s_at, s_stride = row_span("residual_out", residual_out, dtype, index)
        if residual.shape != shape or residual_out.shape != shape:
            raise ValueError("residual and residual_out must have x's shape")
    elif residual_out is not None:
        raise ValueError("residual_out needs a residual")
    if quantize:
        if out is not None:
            raise ValueError("out is not taken with quantize")
        if width % MX_GROUP:
            raise ValueError(f"quantize needs a width that is a multiple of {MX_GROUP}")
        y = mx_empty(shape, x.device)
        values_at, scales_at = y[0].data_ptr(), y[1].data_ptr()
    else:
        y = torch.empty_like(x) if out is None else out
        y_at, y_stride = row_span("out", y, dtype, index)
        if y.shape != shape:
            raise ValueError("out must have x's shape")
    if count:
        a = _lib.VmNormArgs(x_at, r_at or None, w_at, y_at or None, s_at or None, values_at or None, scales_at or None,
                            x_stride, r_stride, y_stride, s_stride, count // width, width, act, weight_act,
                            one_centered, eps)
        _lib.check(device_call(index, _lib.lib().vm_rms_norm, ctypes.byref(a)))
    return y if residual is None else (y, residual_out)


def mx_quantize(x: torch.Tensor) -> MxTensor:
    """x [.., width] bfloat16 or float32 (equally spaced rows, width a multiple of 32 up to 16384) as MX rows."""
    act = _act_dtype("x", x)
    at, stride = row_span("x", x, x.dtype, x.get_device())
    width = x.shape[-1]
    if width % MX_GROUP:
        raise ValueError(f"MX rows need a width that is a multiple of {MX_GROUP}")
    rows = x.numel() // max(width, 1)
    require_32_bits(rows, width)
    y = mx_empty(x.shape, x.device)
    if rows:
        _lib.check(device_call(x.get_device(), _lib.lib().vm_mx_quantize, at, stride, y.values.data_ptr(),
                               y.scales.data_ptr(), rows, width, act))
    return y


__all__ = ["MX_GROUP", "MxTensor", "mx_empty", "mx_quantize", "rms_norm"]
