"""vm_linear at the end of what a grid can hold: refused as unsupported, in front of any launch (no GPU needed)."""
import ctypes

import pytest

from veymoe import _lib

SWIGLU = 1


def _call(rows, k, n, activation, out):
    # addresses of which none is read
    a = _lib.VmLinearArgs(x=1 << 54, weight=1 << 20, out=out, x_stride=k, weight_stride=k, out_stride=n, rows=rows, k=k, n=n,
                          activation=activation)
    return _lib.lib().vm_linear(ctypes.byref(a), None), _lib.last_error()


@pytest.mark.parametrize("rows,k,n,activation", [(1, 4096, 1 << 24, SWIGLU), (4, 1 << 24, 1 << 24, SWIGLU), (2, 3592, 1 << 24, SWIGLU),
                                                 (1 << 28, 8, 1 << 24, 0)])
def test_calls_past_a_grid_are_unsupported(rows, k, n, activation):
    code, message = _call(rows, k, n, activation, 1 << 52)
    assert code == _lib.VM_EUNSUPPORTED and "too large" in message


@pytest.mark.parametrize("rows,k,n,activation", [(1, 4096, (1 << 24) - 2, SWIGLU), (1, 3584, 1 << 24, SWIGLU), (4, 8, 1 << 24, 0),
                                                 (1 << 28, 8, 256, 0), (5, 8, 1 << 24, SWIGLU)])
def test_the_largest_calls_within_one_are_not(rows, k, n, activation):
    """They come as far as the check that their outputs, which lie in the matrix, do not pass."""
    code, message = _call(rows, k, n, activation, (1 << 20) + 16)
    assert code == _lib.VM_EINVAL and "overlaps" in message
