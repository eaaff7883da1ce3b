"""Torch plumbing for the C ABI: device pointers, dtype codes, streams."""
from __future__ import annotations

import ctypes

import torch

from . import _lib

ACT_DTYPES = {torch.bfloat16: _lib.VM_BF16, torch.float32: _lib.VM_F32}
_WORD_DTYPES = (torch.int32, getattr(torch, "uint32", torch.int32))


def shape_of(value):
    return tuple(int(v) for v in value.shape)


def require_device(name: str, tensor, dtypes=None):
    """Check that ``tensor`` is a contiguous tensor on the GPU (optionally of a dtype)."""
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor on the GPU, got {type(tensor).__name__}")
    if not tensor.is_cuda:
        raise TypeError(f"{name} must live on the GPU (got {tensor.device})")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if dtypes is not None and tensor.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {tensor.dtype}; expected one of {dtypes}")
    return tensor


def ptr(tensor) -> int | None:
    if tensor is None:
        return None
    return tensor.data_ptr()


def act_code(tensor) -> int:
    try:
        return ACT_DTYPES[tensor.dtype]
    except KeyError:
        raise TypeError(f"activations must be bfloat16 or float32, got {tensor.dtype}") from None


def word_tensor(name: str, tensor):
    """Route words / packed weights: int32 or uint32 tensors on the GPU."""
    require_device(name, tensor)
    if tensor.dtype not in _WORD_DTYPES:
        raise TypeError(f"{name} must use 32-bit packed values (int32/uint32), got {tensor.dtype}")
    return tensor


def stream_handle(stream=None) -> ctypes.c_void_p:
    if stream is None:
        # the raw handle of torch.cuda.current_stream(), without the Stream
        # object (2.9 us of a call's 20 us on the host)
        return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()))
    return ctypes.c_void_p(stream.cuda_stream)


def device_call(device, call, *args) -> int:
    """``call(*args, stream)`` on ``device``'s current stream, with ``device`` current."""
    if device.index is None or device.index == torch.cuda.current_device():
        return call(*args, stream_handle())
    with torch.cuda.device(device):
        return call(*args, stream_handle())


def rows_view(name: str, tensor, dtypes):
    """``tensor`` [.., width] on the GPU as [rows, width], element stride 1 within a row and one stride between rows;
    a tensor whose rows have no single stride is refused rather than copied."""
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        raise TypeError(f"{name} must be a tensor on the GPU")
    if tensor.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {tensor.dtype}; expected one of {dtypes}")
    if tensor.dim() == 0:
        raise ValueError(f"{name} must have at least one dimension")
    if tensor.dim() != 2:
        try:
            tensor = tensor.view(-1, tensor.shape[-1]) if tensor.numel() else tensor.reshape(-1, tensor.shape[-1])
        except RuntimeError:
            raise ValueError(f"the rows of {name} must have one stride") from None
    if tensor.shape[1] > 1 and tensor.stride(1) != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    return tensor


def row_stride(rows) -> int:
    """Elements between the rows of a [rows, width] view (a single row: its width)."""
    return rows.stride(0) if rows.shape[0] > 1 else max(rows.shape[1], 1)


def require_same_device(device, **tensors):
    for name, tensor in tensors.items():
        if tensor is not None and tensor.device != device:
            raise ValueError(f"{name} is on {tensor.device}, not on {device}")


def route_ids(name: str, ids, count: int):
    """Contiguous int32 group ids on the GPU; 64-bit ids outside 0..count-1 stay outside."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda:
        raise TypeError(f"{name} must be a tensor on the GPU")
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, count).to(torch.int32)
    elif ids.dtype != torch.int32:
        raise TypeError(f"{name} must be int32 or int64, got {ids.dtype}")
    return ids.contiguous()


def q4proj(weight=None, scales=None, biases=None) -> _lib.VmQ4Proj:
    return _lib.VmQ4Proj(ptr(weight), ptr(scales), ptr(biases))


def workspace(nbytes: int, device) -> torch.Tensor:
    """Zero-initialised device scratch (counters in it must start at zero)."""
    return torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)
