"""Products of routed rows with the matrix of their expert, in bf16 or MX.

The Q4 expert block (``grouped.py``, ``HipSwitchGLU``) keeps its weights packed in 4 bits.  ``grouped_matmul`` is the
projection by itself for experts kept in bfloat16 or in MX (``norm.py``): the unquantised counterpart of the
reference's ``gather_qmm`` call (expert_cache.py:818-829, 2017-2037), with the sort by expert, SwiGLU over a gate/up
pair and the 8-bit output for the next product inside the call.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import device_call, require_32_bits, route_ids, row_span
from .norm import MX_GROUP, MxTensor, mx_empty, require_mx


def _matrices(name, w, dtype, index):
    """(address, row stride, expert stride) of a bank [experts, n, k] on GPU ``index`` with contiguous rows."""
    if not isinstance(w, torch.Tensor) or w.dtype != dtype:
        raise TypeError(f"{name} must be a tensor of {dtype}")
    if not w.is_cuda or w.get_device() != index:
        raise TypeError(f"{name} must live on GPU {index} (got {w.device})")
    if w.dim() != 3:
        raise ValueError(f"{name} must have shape (experts, outputs, inputs)")
    expert, row, one = w.stride()
    if one != 1 and w.shape[2] > 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return w.data_ptr(), row, expert


def grouped_matmul(x, weight, inds: torch.Tensor, *, activation: str = None, quantize: bool = False,
                   out: torch.Tensor = None):
    """``x . weight[inds]^T`` for every routed row, sums in fp32.

    weight [experts, n, k] (``activation="swiglu"``: [experts, 2 n, k], gate rows then up rows, and the result is
    silu(gate) * up); inds [tokens, slots] (or any shape) int32/int64 expert ids; x [*inds.shape, k], a row for every
    id, or [*inds.shape[:-1], k], a token's row for all its slots.  x and weight are both bfloat16 tensors (k a
    multiple of 8) or both :class:`MxTensor` (k a multiple of 32); their rows must be 16-byte aligned.  Returns
    [*inds.shape, n] in bfloat16, or as an MxTensor with ``quantize`` (swiglu only, n a multiple of 32).  The row of an
    id outside 0..experts-1 is zero.  Up to 1024 experts.  ``out`` overlaps no operand.  MX values enter as bfloat16:
    those below 2^-126 are rounded to multiples of 2^-133, those of 2^128 and above are infinite.
    """
    mx = isinstance(x, MxTensor)
    if mx != isinstance(weight, MxTensor):
        raise TypeError("x and weight must both be bfloat16 tensors or both be MxTensors")
    if activation not in (None, "swiglu"):
        raise ValueError(f"unknown activation {activation!r}")
    swiglu = activation == "swiglu"
    if quantize and not swiglu:
        raise ValueError("quantize needs the swiglu activation")
    if quantize and out is not None:
        raise ValueError("out is not taken with quantize")
    xv, wv = (require_mx("x", x).values, require_mx("weight", weight).values) if mx else (x, weight)
    dtype = torch.float8_e4m3fn if mx else torch.bfloat16
    index = xv.get_device() if isinstance(xv, torch.Tensor) else None
    x_at, x_stride = row_span("x", xv, dtype, index)
    w_at, w_stride, w_expert = _matrices("weight", wv, dtype, index)
    experts, n, k = wv.shape
    if swiglu:
        if n % 2:
            raise ValueError("swiglu needs an even number of matrix rows (gate, then up)")
        n //= 2
    inds = route_ids("inds", inds, experts, index)
    lead, shape = xv.shape[:-1], inds.shape
    x_div = 1
    if lead != shape:
        if not shape or lead != shape[:-1]:
            raise ValueError(f"x {tuple(xv.shape)} does not fit inds {tuple(shape)} and weight {tuple(wv.shape)}")
        x_div = max(shape[-1], 1)
    if xv.shape[-1] != k:
        raise ValueError(f"x {tuple(xv.shape)} does not fit weight {tuple(wv.shape)}")
    rows = inds.numel()
    require_32_bits(rows, x_div, k, wv.shape[1])
    y_at = values_at = scales_at = None
    if quantize:
        if n % MX_GROUP:
            raise ValueError(f"quantize needs a multiple of {MX_GROUP} outputs")
        y = mx_empty((*shape, n), xv.device)
        values_at, scales_at = y[0].data_ptr(), y[1].data_ptr()
    else:
        if out is None:
            y = torch.empty((*shape, n), dtype=torch.bfloat16, device=xv.device)
        elif not isinstance(out, torch.Tensor):
            raise TypeError(f"out must be a torch tensor, got {type(out).__name__}")
        elif out.shape != (*shape, n) or out.dtype != torch.bfloat16 or not out.is_contiguous() \
                or out.device != xv.device:
            raise ValueError(f"out must be a contiguous bfloat16 tensor of shape {(*shape, n)} on {xv.device}")
        else:
            y = out
        y_at = y.data_ptr()
    if rows == 0 or n == 0:
        return y
    xs_at = ws_at = None
    xs_stride = ws_stride = ws_expert = 0
    if mx:
        xs_at, xs_stride = row_span("x scales", x.scales, x.scales.dtype, index)
        ws_at, ws_stride, ws_expert = _matrices("weight scales", weight.scales, weight.scales.dtype, index)
    lib = _lib.lib()
    nbytes = lib.vm_grouped_matmul_workspace(rows, experts)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=xv.device) if nbytes else None
    a = _lib.VmProductArgs(x_at, xs_at, w_at, ws_at, inds.data_ptr(), y_at, values_at, scales_at,
                           ws.data_ptr() if nbytes else None, nbytes, x_stride, xs_stride, w_stride, w_expert,
                           ws_stride, ws_expert, rows, x_div, k, n, experts, mx, swiglu)
    _lib.check(device_call(index, lib.vm_grouped_matmul, ctypes.byref(a)))
    return y


__all__ = ["grouped_matmul"]
