"""Root-mean-square norm with the residual's addition in front of it, and rows in MX.

MX rows (:class:`MxTensor`) hold e4m3 values with one power-of-two scale (e8m0) per group of 32 along the row: the
least 2^e, e >= -127, that keeps the group's largest magnitude within e4m3's 448, so that no value saturates.  A group
that holds an infinity or a NaN is NaN.  ``grouped_matmul`` multiplies them on the matrix cores, scales included.

The norm is the reference's hc_norm arithmetic (patch_rmsnorm.py:108-135) in fp32 from end to end, rounded once where a
value is stored; the reference has no 8-bit output.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from .device import ACT_DTYPES, device_call, require_same_device, row_stride, rows_view

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
    if not isinstance(t, MxTensor):
        raise TypeError(f"{name} must be an MxTensor")
    if not (t.values.is_cuda and t.scales.is_cuda) or t.values.device != t.scales.device:
        raise TypeError(f"{name} must live on one GPU")
    if t.values.dtype != torch.float8_e4m3fn or t.scales.dtype not in _SCALE_DTYPES:
        raise TypeError(f"{name} must hold float8_e4m3fn values and float8_e8m0fnu (or uint8) scales")
    if t.values.shape[-1] % MX_GROUP or t.scales.shape != (*t.values.shape[:-1], t.values.shape[-1] // MX_GROUP):
        raise ValueError(f"{name} needs one scale per {MX_GROUP} values of a row")
    return t


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor = None,
             one_centered: bool = True, quantize: bool = False, out: torch.Tensor = None,
             residual_out: torch.Tensor = None):
    """``h / sqrt(mean(h^2) + eps) * gain`` over the last dimension, h = x + residual, gain = weight (``one_centered``)
    or 1 + weight.

    x [.., width] bfloat16 or float32 with equally spaced rows, width up to 16384; residual of x's shape and type;
    weight [width] in either type.  Returns the normed rows in x's type, or as an :class:`MxTensor` with ``quantize``
    (width a multiple of 32).  With a residual it returns ``(normed, h)``, h rounded to x's type; the norm itself reads
    the unrounded sum.  ``out`` may be x, ``residual_out`` may be x or residual.
    """
    rows = rows_view("x", x, tuple(ACT_DTYPES))
    width = rows.shape[1]
    device = x.device
    if not isinstance(weight, torch.Tensor) or weight.dtype not in ACT_DTYPES:
        raise TypeError("weight must be a bfloat16 or float32 tensor")
    if weight.shape != (width,) or not weight.is_contiguous():
        raise ValueError(f"weight must be contiguous of shape ({width},)")
    if quantize and out is not None:
        raise ValueError("out is not taken with quantize")
    if residual_out is not None and residual is None:
        raise ValueError("residual_out needs a residual")
    require_same_device(device, weight=weight, residual=residual, out=out, residual_out=residual_out)
    a = _lib.VmNormArgs()
    a.x, a.x_stride = rows.data_ptr(), row_stride(rows)
    a.weight = weight.data_ptr()
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("residual must have x's shape")
        r = rows_view("residual", residual, (x.dtype,))
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=device)
        elif residual_out.shape != x.shape:
            raise ValueError("residual_out must have x's shape")
        s = rows_view("residual_out", residual_out, (x.dtype,))
        a.residual, a.residual_stride = r.data_ptr(), row_stride(r)
        a.sum_out, a.sum_stride = s.data_ptr(), row_stride(s)
    if quantize:
        if width % MX_GROUP:
            raise ValueError(f"quantize needs a width that is a multiple of {MX_GROUP}")
        y = mx_empty(x.shape, device)
        a.values, a.scales = y.values.data_ptr(), y.scales.data_ptr()
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=device) if out is None else out
        if y.shape != x.shape:
            raise ValueError("out must have x's shape")
        o = rows_view("out", y, (x.dtype,))
        a.out, a.out_stride = o.data_ptr(), row_stride(o)
    a.rows, a.width = rows.shape
    a.act_dtype, a.weight_dtype = ACT_DTYPES[x.dtype], ACT_DTYPES[weight.dtype]
    a.one_centered = int(one_centered)
    a.eps = eps
    _lib.check(device_call(device, _lib.lib().vm_rms_norm, ctypes.byref(a)))
    return y if residual is None else (y, residual_out)


def mx_quantize(x: torch.Tensor) -> MxTensor:
    """x [.., width] bfloat16 or float32 (equally spaced rows, width a multiple of 32 up to 16384) as MX rows."""
    rows = rows_view("x", x, tuple(ACT_DTYPES))
    if rows.shape[1] % MX_GROUP:
        raise ValueError(f"MX rows need a width that is a multiple of {MX_GROUP}")
    y = mx_empty(x.shape, x.device)
    _lib.check(device_call(x.device, _lib.lib().vm_mx_quantize, rows.data_ptr(), row_stride(rows),
                           y.values.data_ptr(), y.scales.data_ptr(), rows.shape[0], rows.shape[1],
                           ACT_DTYPES[x.dtype]))
    return y


__all__ = ["MX_GROUP", "MxTensor", "mx_empty", "mx_quantize", "rms_norm"]
