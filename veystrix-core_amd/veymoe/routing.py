"""From a router's logits to experts: softmax or sigmoid scores, a balance bias, groups of experts, top-k, weights.

``router.router_topk`` is the reference's router (softmax over x W^T, top-k, renormalisation) with its product inside the
call.  ``select_experts`` starts from logits (``linear.linear`` with ``dtype=torch.float32`` gives them) and has the
rules of routers that balance their experts without a loss: the bias moves the choice and not the weight, and whole
groups of experts (those of one node) compete before their experts do.  Its ids go into ``products.grouped_matmul`` as
they are, -1 included.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .device import ACT_DTYPES, device_call, require_32_bits, row_span, vector_of

_SCORES = {"softmax": _lib.VM_SCORES_SOFTMAX, "sigmoid": _lib.VM_SCORES_SIGMOID}


def _dtype_code(name, dtype) -> int:
    try:
        return ACT_DTYPES[dtype]
    except KeyError:
        raise TypeError(f"{name} must be bfloat16 or float32, got {dtype}") from None


def select_experts(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: torch.Tensor = None,
                   groups: int = 1, top_groups: int = 1, group_top: int = 1, renormalize: bool = True,
                   scale: float = 1.0, dtype: torch.dtype = torch.float32):
    """``(inds, weights)`` [.., top_k] of logits [.., experts] bfloat16 or float32 (equally spaced rows, up to 1024
    experts; top_k up to 64).

    Scores are the softmax over a row's open experts (logit above -inf) or the sigmoid of each.  The choice is score +
    bias ([experts], bfloat16 or float32), or without a bias the logit itself; it is compared in 64 bits, ties go to the
    lowest index.  With ``groups`` > 1 (up to 64, dividing the experts into ranges of neighbours) only the ``top_groups``
    groups whose ``group_top`` (1 or 2) best choices have the largest sum are chosen from.  Weights are the chosen
    experts' scores without the bias, over their sum with ``renormalize`` (0 where that is 0), times ``scale``, in
    ``dtype`` (float32 or bfloat16).  inds is int32, best first; where a row has no open expert left it holds -1 and
    weight 0.  NaN choices go first, and their weights are NaN.
    """
    if not isinstance(logits, torch.Tensor):
        raise TypeError(f"logits must be a torch tensor on the GPU, got {type(logits).__name__}")
    code, index = _dtype_code("logits", logits.dtype), logits.get_device()
    at, stride = row_span("logits", logits, logits.dtype, index)
    try:
        scores = _SCORES[scoring]
    except (KeyError, TypeError):
        raise ValueError(f"unknown scoring {scoring!r}") from None
    experts = logits.shape[-1]
    rows = logits.numel() // max(experts, 1)
    if not 1 <= top_k <= _lib.VM_SELECT_MAX_TOP_K:
        raise ValueError(f"top_k must be 1..{_lib.VM_SELECT_MAX_TOP_K}")
    if min(groups, top_groups, group_top) < 1:
        raise ValueError("groups, top_groups and group_top must be positive")
    require_32_bits(rows, experts, groups, top_groups, group_top)
    bias_at, bias_code = (None, code) if bias is None else vector_of("bias", bias, experts, index)
    out_code = _dtype_code("dtype", dtype)
    shape, device = (*logits.shape[:-1], top_k), logits.device
    inds = torch.empty(shape, dtype=torch.int32, device=device)
    weights = logits.new_empty(shape) if logits.dtype == dtype else torch.empty(shape, dtype=dtype, device=device)
    a = _lib.VmSelectArgs(at, bias_at, inds.data_ptr(), weights.data_ptr(), stride, scale, rows, experts, groups, top_groups,
                          group_top, top_k, scores, renormalize, code, bias_code, out_code, 0)
    _lib.check(device_call(index, _lib.lib().vm_select_experts, ctypes.byref(a)))
    return inds, weights


__all__ = ["select_experts"]
