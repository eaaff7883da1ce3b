"""Matrix products with bias, activation and residual in their epilogue, bf16 or MX operands.

The dense companion of ``products.grouped_matmul``: shared experts, projections, and with ``dtype=torch.float32`` the
logits that ``routing.select_experts`` takes.  No counterpart in the reference, whose projections are Q4 or plain MLX
products.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import ACT_DTYPES, device_call, require_32_bits, row_span, vector_of
from .norm import MxTensor, require_mx

ACTIVATIONS = {None: _lib.VM_ACTIVATION_NONE, "swiglu": _lib.VM_ACTIVATION_SWIGLU, "relu": _lib.VM_ACTIVATION_RELU,
               "silu": _lib.VM_ACTIVATION_SILU, "gelu": _lib.VM_ACTIVATION_GELU,
               "gelu_tanh": _lib.VM_ACTIVATION_GELU_TANH, "sigmoid": _lib.VM_ACTIVATION_SIGMOID}


def _code(name, t) -> int:
    try:
        return ACT_DTYPES[t.dtype]
    except (AttributeError, KeyError):
        raise TypeError(f"{name} must be a bfloat16 or float32 tensor") from None


def linear(x, weight, bias: torch.Tensor = None, *, activation: str = None, residual: torch.Tensor = None,
           dtype: torch.dtype = torch.bfloat16, out: torch.Tensor = None):
    """``activation(x . weight^T + bias) + residual``, sums and epilogue in fp32, rounded once to ``dtype``.

    x [.., k] and weight [n, k] are both bfloat16 tensors (k a multiple of 8) or both :class:`MxTensor` (k a multiple of
    32); rows equally spaced and 16-byte aligned.  activation: None, "relu", "silu", "gelu" (x Phi(x)), "gelu_tanh",
    "sigmoid", or "swiglu" over a weight (and bias) of 2 n rows, gate then up: silu(gate) * up.  bias contiguous and
    residual [.., n] in bfloat16 or float32; ``dtype`` bfloat16 or float32.  Returns [.., n].  ``out`` [.., n] (of
    ``dtype``, rows equally spaced) may be residual where the types match, and overlaps nothing otherwise.  MX values
    enter as bfloat16: those below 2^-126 are rounded to multiples of 2^-133, those of 2^128 and above are infinite.
    silu, swiglu and sigmoid are off by at most 16 + 2 |x| half steps of fp32, gelu by 12 + 4 x^2, gelu_tanh by 20 + 7 |u|, u
    its sigmoid's argument; where the formula is infinity times zero (silu, gelu, gelu_tanh and swiglu at -infinity) they are
    NaN.
    """
    mx = isinstance(x, MxTensor)
    if mx != isinstance(weight, MxTensor):
        raise TypeError("x and weight must both be bfloat16 tensors or both be MxTensors")
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {activation!r}") from None
    xv, wv = (require_mx("x", x).values, require_mx("weight", weight).values) if mx else (x, weight)
    operand = torch.float8_e4m3fn if mx else torch.bfloat16
    index = xv.get_device() if isinstance(xv, torch.Tensor) else None
    x_at, x_stride = row_span("x", xv, operand, index)
    w_at, w_stride = row_span("weight", wv, operand, index)
    if wv.dim() != 2 or xv.shape[-1] != wv.shape[1]:
        raise ValueError(f"x {tuple(xv.shape)} does not fit weight {tuple(wv.shape)}")
    n, k = wv.shape
    if k == 0:
        raise ValueError("x and weight need at least one input")
    if act == _lib.VM_ACTIVATION_SWIGLU:
        if n % 2:
            raise ValueError("swiglu needs an even number of weight rows (gate, then up)")
        n //= 2
    if dtype not in ACT_DTYPES:
        raise TypeError(f"dtype must be bfloat16 or float32, got {dtype}")
    shape = (*xv.shape[:-1], n)
    rows = xv.numel() // k
    require_32_bits(rows, k, wv.shape[0])
    bias_at = res_at = None
    bias_code = res_code = res_stride = 0
    if bias is not None:
        bias_at, bias_code = vector_of("bias", bias, wv.shape[0], index)
    if residual is not None:
        res_code = _code("residual", residual)
        res_at, res_stride = row_span("residual", residual, residual.dtype, index)
        if residual.shape != shape:
            raise ValueError(f"residual must have shape {shape}")
    if out is None:
        y = xv.new_empty(shape) if xv.dtype == dtype else torch.empty(shape, dtype=dtype, device=xv.device)
        y_at, y_stride = y.data_ptr(), n
    else:
        y = out
        y_at, y_stride = row_span("out", y, dtype, index)
        if y.shape != shape:
            raise ValueError(f"out must have shape {shape}")
    if rows == 0 or n == 0:
        return y
    xs_at = ws_at = None
    xs_stride = ws_stride = 0
    if mx:
        xs_at, xs_stride = row_span("x scales", x.scales, x.scales.dtype, index)
        ws_at, ws_stride = row_span("weight scales", weight.scales, weight.scales.dtype, index)
    a = _lib.VmLinearArgs(x_at, xs_at, w_at, ws_at, bias_at, res_at, y_at, x_stride, xs_stride, w_stride, ws_stride,
                          res_stride, y_stride, rows, k, n, mx, act, bias_code, res_code, ACT_DTYPES[dtype])
    _lib.check(device_call(index, _lib.lib().vm_linear, ctypes.byref(a)))
    return y


__all__ = ["ACTIVATIONS", "linear"]
