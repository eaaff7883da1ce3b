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


_current_device = torch._C._cuda_getDevice


def device_call(index, call, *args) -> int:
    """``call(*args, stream)`` on the current stream of GPU ``index``, with that GPU current."""
    if index == _current_device():
        return call(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return call(*args, torch._C._cuda_getCurrentRawStream(index))


def row_span(name: str, tensor, dtype, index):
    """(address, elements between rows) of the rows of ``tensor`` [.., width], which must be contiguous in themselves,
    lie at one stride (refused rather than copied otherwise), be of ``dtype`` and lie on GPU ``index``."""
    try:
        if tensor.dtype != dtype:
            raise TypeError(f"{name} has dtype {tensor.dtype}; expected {dtype}")
        if not tensor.is_cuda or tensor.get_device() != index:
            raise TypeError(f"{name} must live on GPU {index} (got {tensor.device})")
        strides = tensor.stride()
    except AttributeError:
        raise TypeError(f"{name} must be a torch tensor on the GPU, got {type(tensor).__name__}") from None
    if len(strides) == 2 and strides[1] == 1:
        return tensor.data_ptr(), strides[0]
    shape = tensor.shape
    if not shape:
        raise ValueError(f"{name} must have at least one dimension")
    if shape[-1] > 1 and strides[-1] != 1:
        raise ValueError(f"the rows of {name} must be contiguous")
    step, span = None, 1        # the leading dimensions as one: each stride the inner one's extent
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if step is None:
            step = stride
        elif stride != step * span:
            raise ValueError(f"the rows of {name} must have one stride")
        span *= size
    return tensor.data_ptr(), shape[-1] if step is None else step


def require_32_bits(*sizes):
    """Sizes that the C ABI takes in 32 bits."""
    if max(sizes) >> 32:
        raise ValueError(f"a call takes sizes below 2^32 (got {sizes})")


def route_ids(name: str, ids, count: int, index):
    """Contiguous int32 group ids on GPU ``index``; 64-bit ids outside 0..count-1 stay outside."""
    if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.get_device() != index:
        raise TypeError(f"{name} must be a tensor on GPU {index}")
    if ids.dtype == torch.int64:
        ids = ids.clamp(-1, count).to(torch.int32)
    elif ids.dtype != torch.int32:
        raise TypeError(f"{name} must be int32 or int64, got {ids.dtype}")
    return ids if ids.is_contiguous() else ids.contiguous()


def q4proj(weight=None, scales=None, biases=None) -> _lib.VmQ4Proj:
    return _lib.VmQ4Proj(ptr(weight), ptr(scales), ptr(biases))


def workspace(nbytes: int, device) -> torch.Tensor:
    """Zero-initialised device scratch (counters in it must start at zero)."""
    return torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)
