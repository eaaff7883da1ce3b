"""Root-mean-square norm with the residual's addition in front of it, a block's two norms with its gate and residual, and
rows in MX.

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
from .device import ACT_DTYPES, device_call, require_32_bits, row_span, vector_of

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
    if not isinstance(t, MxTensor) or not isinstance(t[0], torch.Tensor) or not isinstance(t[1], torch.Tensor):
        raise TypeError(f"{name} must be an MxTensor of two tensors")
    values, scales = t
    if values.dtype != torch.float8_e4m3fn or scales.dtype not in _SCALE_DTYPES:
        raise TypeError(f"{name} must hold float8_e4m3fn values and float8_e8m0fnu (or uint8) scales")
    shape, groups = values.shape, scales.shape
    if not shape or not groups or groups[-1] * MX_GROUP != shape[-1] or groups[:-1] != shape[:-1]:
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


def block_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor = None, *, post_weight: torch.Tensor = None,
               gate: torch.Tensor = None, sigmoid_gate: bool = False, scale: float = 1.0, residual_scale: float = 1.0,
               eps: float = 1e-6, one_centered: bool = True, quantize: bool = False, out: torch.Tensor = None,
               residual_out: torch.Tensor = None):
    """From a block's output x to the next block's input: ``(y, h)`` with

        n = x / sqrt(mean(x^2) + eps) * post_weight          (n = x without a post_weight)
        h = residual_scale * residual + scale * gate * n
        y = h / sqrt(mean(h^2) + eps) * weight               (only h is returned without a weight)

    over the last dimension; weights count from zero (1 + weight) unless ``one_centered``.  x [.., width] and residual of
    its shape, each bfloat16 or float32 with equally spaced rows, width up to 16384; weights [width] in either type.
    gate: [.., 1], one for each row, [width], one for each channel, or x's shape, in either type, as it is or with
    ``sigmoid_gate`` through a sigmoid.  h comes in residual's type, y in x's, or as an :class:`MxTensor` with
    ``quantize`` (width a multiple of 32); the second norm reads the unrounded h.  ``out`` and ``residual_out`` may each
    be x or residual where the types match, and overlap nothing otherwise.
    """
    act, res_act = _act_dtype("x", x), _act_dtype("residual", residual)
    shape, index = x.shape, x.get_device()
    x_at, x_stride = row_span("x", x, x.dtype, index)
    r_at, r_stride = row_span("residual", residual, residual.dtype, index)
    if residual.shape != shape:
        raise ValueError("residual must have x's shape")
    width, count = shape[-1], x.numel()
    rows = count // width if count else 0
    require_32_bits(rows, width)
    post_at = w_at = gate_at = None
    post_code = w_code = gate_code = gate_stride = 0
    kind = _lib.VM_GATE_NONE
    if post_weight is not None:
        post_at, post_code = vector_of("post_weight", post_weight, width, index)
    if weight is not None:
        w_at, w_code = vector_of("weight", weight, width, index)
    elif quantize or out is not None:
        raise ValueError("quantize and out need a weight")
    if gate is not None:
        gate_code = _act_dtype("gate", gate)
        gate_at, gate_stride = row_span("gate", gate, gate.dtype, index)
        if gate.shape == shape and len(shape) > 1:
            kind = _lib.VM_GATE_VALUE
        elif gate.shape == (width,):
            kind = _lib.VM_GATE_CHANNEL
        elif gate.shape == (*shape[:-1], 1):
            kind = _lib.VM_GATE_ROW
        else:
            raise ValueError(f"gate {tuple(gate.shape)} is neither one per row, per channel nor per value of x {tuple(shape)}")
    if quantize:
        if out is not None:
            raise ValueError("out is not taken with quantize")
        if width % MX_GROUP:
            raise ValueError(f"quantize needs a width that is a multiple of {MX_GROUP}")
    if residual_out is None:
        h = torch.empty_like(residual)
        h_at, h_stride = (h.data_ptr(), width) if h.is_contiguous() else row_span("residual", h, h.dtype, index)
    else:
        h = residual_out
        h_at, h_stride = row_span("residual_out", h, residual.dtype, index)
        if h.shape != shape:
            raise ValueError("residual_out must have x's shape")
    y = y_at = values_at = scales_at = None
    y_stride = 0
    if quantize:
        y = mx_empty(shape, x.device)
        values_at, scales_at = y[0].data_ptr(), y[1].data_ptr()
    elif out is not None:
        y = out
        y_at, y_stride = row_span("out", y, x.dtype, index)
        if y.shape != shape:
            raise ValueError("out must have x's shape")
    elif weight is not None:
        y = torch.empty_like(x)
        y_at, y_stride = (y.data_ptr(), width) if y.is_contiguous() else row_span("x", y, y.dtype, index)
    if rows:
        a = _lib.VmBlockNormArgs(x_at, r_at, post_at, gate_at, w_at, y_at, h_at, values_at, scales_at, x_stride, r_stride,
                                 gate_stride, y_stride, h_stride, scale, residual_scale, eps, rows, width, act, res_act,
                                 post_code, gate_code, w_code, kind, sigmoid_gate, one_centered)
        _lib.check(device_call(index, _lib.lib().vm_block_norm, ctypes.byref(a)))
    return h if weight is None else (y, h)


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


__all__ = ["MX_GROUP", "MxTensor", "block_norm", "mx_empty", "mx_quantize", "rms_norm"]
