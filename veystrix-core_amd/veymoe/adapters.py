"""Low-rank adapters of many requests at once, beside the projection that they share.

A batch mixes requests whose projections differ by a low-rank term of their own.  The shared projection runs once for
all rows; ``add_adapters`` adds every row's ``scale * B (A x)`` to its output.  The reference serves one request at a
time and has no adapters.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import device_call, require_same_device, route_ids, row_stride, rows_view

_BF16 = (torch.bfloat16,)


def _bank(name, t, shape):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be a bfloat16 tensor")
    if t.dim() != 3 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous of shape {shape}")


def add_adapters(base: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, *,
                 scales: torch.Tensor = None, out: torch.Tensor = None) -> torch.Tensor:
    """``base + scales[i] * b[i] (a[i] x)`` per row, i = ids of the row; base where ids names no adapter.

    base [.., n] the shared projection's output and x [.., k] its input, bfloat16 with equally spaced rows; a
    [adapters, rank, k] and b [adapters, n, rank] bfloat16, contiguous; ids [..] int32/int64; scales [adapters] float32
    (1 without).  Up to 1024 adapters of rank up to 128.  The rank sums stay in fp32, and the result is rounded once.
    ``out`` may be base.
    """
    x_rows, base_rows = rows_view("x", x, _BF16), rows_view("base", base, _BF16)
    _bank("a", a, "(adapters, rank, k)")
    _bank("b", b, "(adapters, n, rank)")
    adapters, rank, k = a.shape
    n = base_rows.shape[1]
    if x_rows.shape[1] != k or tuple(b.shape) != (adapters, n, rank) or x.shape[:-1] != base.shape[:-1]:
        raise ValueError(f"base {tuple(base.shape)}, x {tuple(x.shape)}, a {tuple(a.shape)} and b {tuple(b.shape)} "
                         "do not fit together")
    ids = route_ids("ids", ids, adapters)
    if ids.shape != x.shape[:-1]:
        raise ValueError(f"ids must have shape {tuple(x.shape[:-1])}")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (adapters,)
                               or not scales.is_contiguous()):
        raise ValueError(f"scales must be contiguous float32 of shape ({adapters},)")
    device = x.device
    if out is None:
        out = torch.empty(base.shape, dtype=base.dtype, device=device)
    elif out.shape != base.shape:
        raise ValueError("out must have base's shape")
    require_same_device(device, base=base, a=a, b=b, ids=ids, scales=scales, out=out)
    out_rows = rows_view("out", out, _BF16)
    if out.numel() == 0:
        return out
    p = _lib.VmAdapterArgs()
    p.base, p.base_stride = base_rows.data_ptr(), row_stride(base_rows)
    p.x, p.x_stride = x_rows.data_ptr(), row_stride(x_rows)
    p.out, p.out_stride = out_rows.data_ptr(), row_stride(out_rows)
    p.a, p.b, p.ids = a.data_ptr(), b.data_ptr(), ids.data_ptr()
    if scales is not None:
        p.scales = scales.data_ptr()
    rows = x_rows.shape[0]
    p.rows, p.k, p.n, p.rank, p.adapters = rows, k, n, rank, adapters
    lib = _lib.lib()
    nbytes = lib.vm_add_adapters_workspace(rows, adapters)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    _lib.check(device_call(device, lib.vm_add_adapters, ctypes.byref(p)))
    return out


__all__ = ["add_adapters"]
