"""Arguments of the norm, the products and the adapters that are no tensors: TypeError, as for tensors of a wrong type."""
import numpy as np
import pytest
import torch

from veymoe.adapters import add_adapters
from veymoe.norm import MxTensor, mx_quantize, rms_norm
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wrong", [0.5, [1.0], "x", np.zeros((4, 64), np.float32)], ids=["number", "list", "text", "array"])
def test_arguments_that_are_no_tensors(device, wrong):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    g = torch.ones(64, dtype=torch.bfloat16, device=device)
    w = torch.zeros((3, 32, 64), dtype=torch.bfloat16, device=device)
    inds = torch.zeros((4, 2), dtype=torch.int32, device=device)
    a, b, ids = w[:, :8].contiguous(), torch.zeros((3, 64, 8), dtype=torch.bfloat16, device=device), inds[:, 0].contiguous()
    qx, qw = mx_quantize(x), mx_quantize(w)
    calls = [lambda: rms_norm(wrong, g), lambda: rms_norm(x, wrong), lambda: rms_norm(x, g, residual=wrong),
             lambda: rms_norm(x, g, residual=x, residual_out=wrong), lambda: rms_norm(x, g, out=wrong),
             lambda: mx_quantize(wrong), lambda: grouped_matmul(wrong, w, inds), lambda: grouped_matmul(x, wrong, inds),
             lambda: grouped_matmul(x, w, wrong), lambda: grouped_matmul(x, w, inds, out=wrong),
             lambda: grouped_matmul(MxTensor(wrong, qx.scales), qw, inds),
             lambda: grouped_matmul(qx, MxTensor(qw.values, wrong), inds),
             lambda: add_adapters(wrong, x, a, b, ids), lambda: add_adapters(x, wrong, a, b, ids),
             lambda: add_adapters(x, x, wrong, b, ids), lambda: add_adapters(x, x, a, wrong, ids),
             lambda: add_adapters(x, x, a, b, wrong), lambda: add_adapters(x, x, a, b, ids, out=wrong)]
    for n, call in enumerate(calls):
        try:
            call()
        except TypeError:
            continue
        except Exception as e:  # noqa: BLE001
            pytest.fail(f"call {n}: {type(e).__name__}: {e}")
        pytest.fail(f"call {n} took {wrong!r}")
