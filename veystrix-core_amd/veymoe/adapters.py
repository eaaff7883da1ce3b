"""Low-rank adapters of many requests at once, beside the projection that they share.

A batch mixes requests whose projections differ by a low-rank term of their own.  The shared projection runs once for
all rows; ``add_adapters`` adds every row's ``scale * B (A x)`` to its output.  The reference serves one request at a
time and has no adapters.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import device_call, require_32_bits, route_ids, row_span

_BF16 = torch.bfloat16


def _bank(name, t, index):
    if not isinstance(t, torch.Tensor) or t.dtype != _BF16 or not t.is_cuda or t.get_device() != index:
        raise TypeError(f"{name} must be a bfloat16 tensor on GPU {index}")
    if t.dim() != 3 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bank of matrices")
    return t.data_ptr()


def add_adapters(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, *,
                 scales: torch.Tensor = None, out: torch.Tensor = None) -> torch.Tensor:
    """``base + scales[i] * b[i] (a[i] x)`` per row, i = ids of the row; base where ids names no adapter.

    base [.., n] the shared projection's output and x [.., k] its input, bfloat16 with equally spaced rows; a
    [adapters, rank, k] and b [adapters, n, rank] bfloat16, contiguous; ids [..] int32/int64; scales [adapters] float32
    (1 without).  Up to 1024 adapters of rank up to 128.  The rank sums stay in fp32, and the result is rounded once.
    ``out`` may be base, and overlaps nothing otherwise.
    """
    index = x.get_device() if isinstance(x, torch.Tensor) else None
    x_at, x_stride = row_span("x", x, _BF16, index)
    base_at, base_stride = row_span("base", base, _BF16, index)
    a_at, b_at = _bank("a", a, index), _bank("b", b, index)
    adapters, rank, k = a.shape
    lead, shape = x.shape[:-1], base.shape
    n = shape[-1]
    if x.shape[-1] != k or b.shape != (adapters, n, rank) or lead != shape[:-1]:
        raise ValueError(f"base {tuple(shape)}, x {tuple(x.shape)}, a {tuple(a.shape)} and b {tuple(b.shape)} "
                         "do not fit together")
    ids = route_ids("ids", ids, adapters, index)
    if ids.shape != lead:
        raise ValueError(f"ids must have shape {tuple(lead)}")
    rows = ids.numel()
    require_32_bits(rows, k, n, rank)
    scales_at = None
    if scales is not None:
        if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or scales.shape != (adapters,) \
                or not scales.is_contiguous() or scales.device != x.device:
            raise ValueError(f"scales must be contiguous float32 of shape ({adapters},) on {x.device}")
        scales_at = scales.data_ptr()
    if out is None:
        out = torch.empty_like(base)
    out_at, out_stride = row_span("out", out, _BF16, index)
    if out.shape != shape:
        raise ValueError("out must have base's shape")
    if rows == 0 or n == 0:
        return out
    lib = _lib.lib()
    nbytes = lib.vm_add_adapters_workspace(rows, rank, adapters)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    p = _lib.VmAdapterArgs(base_at, x_at, a_at, b_at, scales_at, ids.data_ptr(), out_at,
                           ws.data_ptr() if nbytes else None, nbytes, base_stride, x_stride, out_stride, rows, k, n,
                           rank, adapters)
    _lib.check(device_call(index, lib.vm_add_adapters, ctypes.byref(p)))
    return out


__all__ = ["add_adapters"]
