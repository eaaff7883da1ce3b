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
from .device import device_call, require_same_device, route_ids, row_stride, rows_view
from .norm import MX_GROUP, MxTensor, mx_empty, require_mx


def _matrices(name, w):
    """(row stride, expert stride) of weight [experts, n, k] with contiguous rows."""
    if w.dim() != 3:
        raise ValueError(f"{name} must have shape (experts, outputs, inputs)")
    if w.shape[2] > 1 and w.stride(2) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return (w.stride(1) if w.shape[1] > 1 else w.shape[2]), (w.stride(0) if w.shape[0] > 1 else 0)


def grouped_matmul(x, weight, inds: torch.Tensor, *, activation: str = None, quantize: bool = False,
                   out: torch.Tensor = None):
    """``x . weight[inds]^T`` for every routed row, sums in fp32.

    weight [experts, n, k] (``activation="swiglu"``: [experts, 2 n, k], gate rows then up rows, and the result is
    silu(gate) * up); inds [tokens, slots] (or any shape) int32/int64 expert ids; x [*inds.shape, k], a row for every
    id, or [*inds.shape[:-1], k], a token's row for all its slots.  x and weight are both bfloat16 tensors (k a
    multiple of 8) or both :class:`MxTensor` (k a multiple of 32); their rows must be 16-byte aligned.  Returns
    [*inds.shape, n] in bfloat16, or as an MxTensor with ``quantize`` (swiglu only, n a multiple of 32).  The row of an
    id outside 0..experts-1 is zero.  Up to 1024 experts.
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
    if not isinstance(wv, torch.Tensor) or not wv.is_cuda:
        raise TypeError("weight must be a tensor on the GPU")
    if not mx and wv.dtype != torch.bfloat16:
        raise TypeError(f"weight has dtype {wv.dtype}; expected bfloat16 or an MxTensor")
    rows = rows_view("x", xv, (torch.float8_e4m3fn if mx else torch.bfloat16,))
    device = rows.device
    a = _lib.VmProductArgs()
    a.weight_stride, a.weight_expert_stride = _matrices("weight", wv)
    experts, matrix, k = wv.shape
    if swiglu and matrix % 2:
        raise ValueError("swiglu needs an even number of matrix rows (gate, then up)")
    n = matrix // 2 if swiglu else matrix
    inds = route_ids("inds", inds, experts)
    shape = tuple(inds.shape)
    if tuple(xv.shape) == (*shape, k):
        x_div = 1
    elif shape and tuple(xv.shape) == (*shape[:-1], k):
        x_div = shape[-1]
    else:
        raise ValueError(f"x of shape {tuple(xv.shape)} does not fit inds {shape} and weight {tuple(wv.shape)}")
    require_same_device(device, weight=wv, inds=inds, out=out)
    if quantize:
        if n % MX_GROUP:
            raise ValueError(f"quantize needs a multiple of {MX_GROUP} outputs")
        y = mx_empty((*shape, n), device)
        a.out_values, a.out_scales = y.values.data_ptr(), y.scales.data_ptr()
    else:
        y = torch.empty((*shape, n), dtype=torch.bfloat16, device=device) if out is None else out
        if y.shape != (*shape, n) or y.dtype != torch.bfloat16 or not y.is_contiguous():
            raise ValueError(f"out must be a contiguous bfloat16 tensor of shape {(*shape, n)}")
        a.out = y.data_ptr()
    count = inds.numel()
    if count == 0 or n == 0:
        return y
    a.x, a.x_stride = rows.data_ptr(), row_stride(rows)
    a.weight = wv.data_ptr()
    if mx:
        scales = rows_view("x scales", x.scales, (x.scales.dtype,))
        a.x_scales, a.x_scale_stride = scales.data_ptr(), row_stride(scales)
        a.weight_scales = weight.scales.data_ptr()
        a.weight_scale_stride, a.weight_scale_expert_stride = _matrices("weight scales", weight.scales)
        a.format = _lib.VM_FORMAT_MX
    a.ids = inds.data_ptr()
    a.rows, a.x_div, a.k, a.n, a.experts = count, x_div, k, n, experts
    a.activation = int(swiglu)
    lib = _lib.lib()
    nbytes = lib.vm_grouped_matmul_workspace(count, experts)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    _lib.check(device_call(device, lib.vm_grouped_matmul, ctypes.byref(a)))
    return y


__all__ = ["grouped_matmul"]
