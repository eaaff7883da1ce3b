"""What select_experts, block_norm and linear refuse: arguments that are no tensors or of a wrong type, shape or place."""
import numpy as np
import pytest
import torch

from veymoe.linear import linear
from veymoe.norm import MxTensor, block_norm, mx_quantize
from veymoe.routing import select_experts

pytestmark = pytest.mark.gpu


def _raises(kind, calls):
    for n, call in enumerate(calls):
        try:
            call()
        except kind:
            continue
        except Exception as e:  # noqa: BLE001
            pytest.fail(f"call {n}: {type(e).__name__}: {e}")
        pytest.fail(f"call {n} was taken")


@pytest.mark.parametrize("wrong", [0.5, [1.0], "x", np.zeros((4, 64), np.float32), torch.zeros((4, 64)), torch.zeros(64)],
                         ids=["number", "list", "text", "array", "cpu", "cpu vector"])
def test_arguments_of_a_wrong_kind(device, wrong):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    g, w = torch.ones(64, dtype=torch.bfloat16, device=device), torch.zeros((32, 64), dtype=torch.bfloat16, device=device)
    qx, qw = mx_quantize(x), mx_quantize(w)
    half = torch.zeros((4, 64), dtype=torch.float16, device=device)
    whole = torch.zeros((4, 64), dtype=torch.int32, device=device)
    _raises(TypeError, [
        lambda: select_experts(wrong, 2), lambda: select_experts(x, 2, bias=wrong), lambda: select_experts(half, 2),
        lambda: select_experts(whole, 2), lambda: select_experts(x, 2, bias=half[0]), lambda: select_experts(x, 2, dtype=torch.float16),
        lambda: block_norm(wrong, x, g), lambda: block_norm(x, wrong, g), lambda: block_norm(x, x, wrong),
        lambda: block_norm(x, x, g, post_weight=wrong), lambda: block_norm(x, x, g, gate=wrong),
        lambda: block_norm(x, x, g, out=wrong), lambda: block_norm(x, x, g, residual_out=wrong), lambda: block_norm(half, x, g),
        lambda: block_norm(x, half, g), lambda: block_norm(x, x, g, gate=half), lambda: block_norm(x, x, half[0]),
        lambda: block_norm(x, x, g, out=x.float()), lambda: block_norm(x, x, g, residual_out=x.float()),
        lambda: linear(wrong, w), lambda: linear(x, wrong), lambda: linear(x, w, wrong), lambda: linear(x, w, residual=wrong),
        lambda: linear(x, w, out=wrong), lambda: linear(qx, w), lambda: linear(x, qw), lambda: linear(MxTensor(wrong, qx.scales), qw),
        lambda: linear(qx, MxTensor(qw.values, wrong)), lambda: linear(x.float(), w), lambda: linear(x, w.float()),
        lambda: linear(x, w, half[0, :32]), lambda: linear(x, w, residual=half[:, :32]), lambda: linear(x, w, dtype=torch.float16),
        lambda: linear(x, w, out=x.float()[:, :32])])


def test_arguments_of_a_wrong_shape_or_value(device):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=device)
    g, w = torch.ones(64, dtype=torch.bfloat16, device=device), torch.zeros((32, 64), dtype=torch.bfloat16, device=device)
    y = torch.zeros((4, 32), dtype=torch.bfloat16, device=device)
    odd = torch.zeros((4, 72), dtype=torch.bfloat16, device=device)
    from veymoe import _lib

    _raises((ValueError, _lib.VeymoeError), [
        lambda: select_experts(x, 0), lambda: select_experts(x, 65), lambda: select_experts(x, -1),
        lambda: select_experts(x, 9, groups=8), lambda: select_experts(x, 2, groups=7), lambda: select_experts(x, 2, groups=0),
        lambda: select_experts(x, 2, groups=4, top_groups=5), lambda: select_experts(x, 2, group_top=3),
        lambda: select_experts(x, 2, scoring="relu"), lambda: select_experts(x, 2, scoring=[]),
        lambda: select_experts(x, 2, bias=g[:63]), lambda: select_experts(x, 2, bias=odd[0, ::2]),
        lambda: select_experts(x.t(), 2), lambda: select_experts(torch.zeros((2, 1025), device=device), 2),
        lambda: block_norm(x, x[:3], g), lambda: block_norm(x, x, g[:63]), lambda: block_norm(x, x, g, post_weight=g[:32]),
        lambda: block_norm(x, x, g, gate=x[:3]), lambda: block_norm(x, x, g, gate=g[:32]), lambda: block_norm(x, x, g, out=odd),
        lambda: block_norm(x, x, g, residual_out=odd), lambda: block_norm(x, x, quantize=True), lambda: block_norm(x, x, out=x),
        lambda: block_norm(x, x, g, quantize=True, out=x), lambda: block_norm(odd, odd, torch.ones(72, device=device), quantize=True),
        lambda: block_norm(x.t(), x.t(), g[:4]), lambda: block_norm(x, x, g, out=g.expand(4, 64)),
        lambda: block_norm(torch.zeros((2, 16385), device=device), torch.zeros((2, 16385), device=device)),
        lambda: linear(x, w[:, :32]), lambda: linear(x, w[0]), lambda: linear(x[:, :60], w[:, :60]), lambda: linear(x, w, g),
        lambda: linear(x, w, residual=x), lambda: linear(x, w, out=x), lambda: linear(x, w[:31], activation="swiglu"),
        lambda: linear(x, w, activation="tanh"), lambda: linear(x, w, activation=[]), lambda: linear(x[:, 1:57], w[:, :56]),
        lambda: linear(odd[:, :56][:, ::1], w[:, 4:60]), lambda: linear(x[:, :0], w[:, :0]), lambda: linear(x, w, out=x[:, :32]),
        lambda: linear(x, w, out=w[:4, :32]), lambda: linear(x, w, out=y, residual=odd[:3, :32]),
        lambda: linear(torch.zeros((4, 68), dtype=torch.bfloat16, device=device)[:, :64], w)])
