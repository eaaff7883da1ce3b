"""The argument checks of vm_rms_norm, vm_mx_quantize, vm_grouped_matmul and vm_add_adapters, which reject bad calls
before touching a device, and the layouts of their argument structures (no GPU needed)."""
import ctypes
import os
import subprocess

import pytest

from veymoe import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "veymoe.h")


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"VmNormArgs": _lib.VmNormArgs, "VmProductArgs": _lib.VmProductArgs, "VmAdapterArgs": _lib.VmAdapterArgs}
    constants = ("VM_FORMAT_BF16", "VM_FORMAT_MX", "VM_ACTIVATION_NONE", "VM_ACTIVATION_SWIGLU", "VM_MX_GROUP",
                 "VM_NORM_MAX_WIDTH", "VM_PRODUCT_MAX_EXPERTS", "VM_ADAPTER_MAX_RANK")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines += [f'printf("{c} %u\\n", (unsigned){c});' for c in constants] + ["return 0; }"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    values = dict(line.rsplit(" ", 1) for line in out if line)
    for name, cls in structs.items():
        assert int(values[name]) == ctypes.sizeof(cls), name
        for field, _ in cls._fields_:
            assert int(values[f"{name}.{field}"]) == getattr(cls, field).offset, (name, field)
    for c in constants:
        assert int(values[c]) == getattr(_lib, c), c


def _norm(**kw):
    a = _lib.VmNormArgs()
    a.x, a.weight, a.out = 4096, 8192, 12288
    a.x_stride = a.out_stride = a.sum_stride = a.residual_stride = 64
    a.rows, a.width, a.eps = 2, 64, 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().vm_rms_norm(ctypes.byref(a), None)


@pytest.mark.parametrize("fields,code,message", [
    ({"act_dtype": 2}, _lib.VM_EINVAL, "dtypes"),
    ({"weight_dtype": 5}, _lib.VM_EINVAL, "dtypes"),
    ({"width": 0}, _lib.VM_EUNSUPPORTED, "width"),
    ({"width": 16385}, _lib.VM_EUNSUPPORTED, "width"),
    ({"rows": 1 << 24}, _lib.VM_EUNSUPPORTED, "rows"),
    ({"x": None}, _lib.VM_EINVAL, "required"),
    ({"weight": None}, _lib.VM_EINVAL, "required"),
    ({"out": None}, _lib.VM_EINVAL, "either out"),
    ({"values": 64, "scales": 64}, _lib.VM_EINVAL, "either out"),
    ({"out": None, "values": 64}, _lib.VM_EINVAL, "both values and scales"),
    ({"out": None, "values": 64, "scales": 64, "width": 48}, _lib.VM_EINVAL, "multiple of 32"),
    ({"out": None, "values": 68, "scales": 64}, _lib.VM_EINVAL, "8-byte"),
    ({"out_stride": 63}, _lib.VM_EINVAL, "strides of outputs"),
    ({"sum_out": 4096, "sum_stride": 0}, _lib.VM_EINVAL, "strides of outputs"),
])
def test_norm_rejects(fields, code, message):
    assert _norm(**fields) == code
    assert message in _lib.last_error()


def test_norm_and_quantize_of_nothing():
    assert _norm(rows=0) == _lib.VM_OK
    lib = _lib.lib()
    assert lib.vm_rms_norm(None, None) == _lib.VM_EINVAL
    assert lib.vm_mx_quantize(None, 0, None, None, 0, 32, 0, None) == _lib.VM_OK
    assert lib.vm_mx_quantize(None, 32, 64, 64, 1, 32, 0, None) == _lib.VM_EINVAL
    assert lib.vm_mx_quantize(4096, 40, 64, 64, 1, 40, 0, None) == _lib.VM_EINVAL
    assert lib.vm_mx_quantize(4096, 32, None, 64, 1, 32, 0, None) == _lib.VM_EINVAL
    assert lib.vm_mx_quantize(4096, 32, 64, 64, 1, 32, 2, None) == _lib.VM_EINVAL


def _product(**kw):
    a = _lib.VmProductArgs()
    a.x, a.weight, a.ids, a.out = 4096, 8192, 12288, 16384
    a.x_stride = a.weight_stride = 64
    a.weight_expert_stride = 64 * 32
    a.rows, a.x_div, a.k, a.n, a.experts = 2, 1, 64, 32, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().vm_grouped_matmul(ctypes.byref(a), None)


MX = {"format": _lib.VM_FORMAT_MX, "x_scales": 64, "weight_scales": 64}


@pytest.mark.parametrize("fields,code,message", [
    ({"format": 2}, _lib.VM_EINVAL, "format"),
    ({"activation": 2}, _lib.VM_EINVAL, "activation"),
    ({"k": 0}, _lib.VM_EINVAL, "positive"),
    ({"n": 0}, _lib.VM_EINVAL, "positive"),
    ({"k": 60}, _lib.VM_EUNSUPPORTED, "multiple of 8"),
    ({**MX, "k": 48}, _lib.VM_EUNSUPPORTED, "multiple of 32"),
    ({"experts": 0}, _lib.VM_EUNSUPPORTED, "experts"),
    ({"experts": 1025}, _lib.VM_EUNSUPPORTED, "experts"),
    ({"x_div": 0}, _lib.VM_EINVAL, "x_div"),
    ({"rows": (1 << 28) + 1}, _lib.VM_EUNSUPPORTED, "2^28"),
    ({"x": None}, _lib.VM_EINVAL, "required"),
    ({"ids": None}, _lib.VM_EINVAL, "required"),
    ({**MX, "x_scales": None}, _lib.VM_EINVAL, "x_scales"),
    ({"out": None}, _lib.VM_EINVAL, "either out"),
    ({"out_values": 64}, _lib.VM_EINVAL, "either out"),
    ({"out": None, "out_values": 64, "out_scales": 64}, _lib.VM_EUNSUPPORTED, "swiglu"),
    ({"out": None, "out_values": 64, "out_scales": 64, "activation": 1, "n": 48}, _lib.VM_EINVAL, "multiple of 32"),
    ({"out": None, "out_values": 64, "activation": 1}, _lib.VM_EINVAL, "both values and scales"),
    ({"x": 4104}, _lib.VM_EINVAL, "16-byte"),
    ({"x_stride": 68}, _lib.VM_EINVAL, "16-byte"),
    ({"weight_stride": 68}, _lib.VM_EINVAL, "16-byte"),
    ({"weight_expert_stride": 2052}, _lib.VM_EINVAL, "16-byte"),
    ({"rows": 5000}, _lib.VM_EWORKSPACE, "workspace"),
    ({"rows": 5000, "workspace": 264, "workspace_bytes": 1 << 30}, _lib.VM_EWORKSPACE, "aligned"),
    ({"rows": 1 << 28, "n": 1 << 24}, _lib.VM_EUNSUPPORTED, "too large"),
])
def test_product_rejects(fields, code, message):
    assert _product(**fields) == code
    assert message in _lib.last_error()


def test_product_of_nothing_and_workspace():
    lib = _lib.lib()
    assert _product(rows=0) == _lib.VM_OK
    assert lib.vm_grouped_matmul(None, None) == _lib.VM_EINVAL
    assert lib.vm_grouped_matmul_workspace(1, 512) == 0                       # rows one by one: no sort
    assert lib.vm_grouped_matmul_workspace(4096, 512) >= 4096 * 4 


def _adapters(**kw):
    a = _lib.VmAdapterArgs()
    a.base, a.x, a.a, a.b, a.ids, a.out = 4096, 8192, 12288, 16384, 20480, 24576
    a.base_stride, a.x_stride, a.out_stride = 32, 64, 32
    a.rows, a.k, a.n, a.rank, a.adapters = 2, 64, 32, 8, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().vm_add_adapters(ctypes.byref(a), None)


@pytest.mark.parametrize("fields,code,message", [
    ({"k": 0}, _lib.VM_EINVAL, "k and n"),
    ({"n": (1 << 24) + 1}, _lib.VM_EINVAL, "k and n"),
    ({"rank": 0}, _lib.VM_EUNSUPPORTED, "rank"),
    ({"rank": 129}, _lib.VM_EUNSUPPORTED, "rank"),
    ({"adapters": 1025}, _lib.VM_EUNSUPPORTED, "adapters"),
    ({"base": None}, _lib.VM_EINVAL, "required"),
    ({"out": None}, _lib.VM_EINVAL, "required"),
    ({"out_stride": 31}, _lib.VM_EINVAL, "stride of out"),
    ({"out": 4096, "out_stride": 40}, _lib.VM_EINVAL, "in place"),
    ({"rows": 5000}, _lib.VM_EWORKSPACE, "workspace"),
    ({"rows": 1 << 30}, _lib.VM_EUNSUPPORTED, "too large"),
])
def test_adapters_rejects(fields, code, message):
    assert _adapters(**fields) == code
    assert message in _lib.last_error()


def test_adapters_of_nothing():
    assert _adapters(rows=0) == _lib.VM_OK
    assert _lib.lib().vm_add_adapters(None, None) == _lib.VM_EINVAL


# x at 1 << 20, two rows of 128 bytes; the other arrays of the helpers lie below it
APART = 1 << 20


@pytest.mark.parametrize("fields", [
    {"out": 4096 + 2},                                               # x a value further
    {"out": 4096, "out_stride": 72},                                 # x at another stride
    {"x": APART, "out": APART + 100, "out_stride": 128, "x_stride": 128},
    {"out": 8192},                                                   # weight
    {"out": 8192 - 128},                                             # its second row is the weight
    {"residual": APART, "out": APART + 128},                         # residual's second row
    {"residual": APART, "sum_out": 12288},                           # sum_out is out
    {"residual": APART, "sum_out": 4096 + 64},
    {"residual": APART, "sum_out": APART + 64},
    {"residual": APART, "sum_out": 8192 + 64},
    {"out": None, "values": 4096 + 64, "scales": 1 << 21},
    {"out": None, "values": 1 << 21, "scales": 8192},
    {"out": None, "values": 1 << 21, "scales": 1 << 22, "residual": APART, "sum_out": (1 << 21) + 64},
])
def test_norm_rejects_outputs_over_operands(fields):
    assert _norm(**fields) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("fields", [
    {"out": 4096}, {"out": 4096 + 127}, {"out": 8192}, {"out": 8192 + 4 * 32 * 128 - 2}, {"out": 12288 + 4},
    {"out": 12288 - 64},                                             # its second row
    {**MX, "x_scales": 1 << 21, "weight_scales": 1 << 22, "out": (1 << 21) + 2, "x_scale_stride": 2},
    {"activation": 1, "out": None, "out_values": 4096 + 64, "out_scales": 1 << 21},
    {"activation": 1, "out": None, "out_values": 1 << 21, "out_scales": 8192 + 2},
])
def test_product_rejects_outputs_over_operands(fields):
    assert _product(**fields) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("fields", [
    {"out": 4096 + 2}, {"out": 4096 + 64}, {"out": 8192}, {"out": 8192 + 32, "out_stride": 64}, {"out": 12288}, {"out": 16384},
    {"out": 20480}, {"scales": 24576 + 8},
])
def test_adapters_reject_outputs_over_operands(fields):
    assert _adapters(**fields) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("values,scales,x_stride", [(APART, 64, 64), (APART + 64, 64, 64), (APART - 120, 64, 64),
                                                    (64, APART + 127, 64), (64, APART - 3, 64), (APART + 256, 64, 128)])
def test_quantize_rejects_outputs_over_its_input(values, scales, x_stride):
    """x: two bf16 rows of 64 at APART; rows of another stride are no way past it."""
    lib = _lib.lib()
    assert lib.vm_mx_quantize(APART, x_stride, values, scales, 2, 64, 0, None) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("scales", [APART, APART + 127, APART - 3])
def test_values_over_scales_are_rejected(scales):
    """Two rows of 64 values at APART, two scales each."""
    lib = _lib.lib()
    assert lib.vm_mx_quantize(4096, 64, APART, scales, 2, 64, 0, None) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()
    assert _norm(out=None, values=APART, scales=scales) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()
    # n = 64: a gate/up bank of 4 x 128 rows of 64
    assert _product(x=1 << 24, weight=1 << 25, weight_expert_stride=64 * 128, n=64, activation=1, out=None,
                    out_values=APART, out_scales=scales) == _lib.VM_EINVAL
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("over", ["x", "weight", "ids", "out"])
def test_product_rejects_a_workspace_over_its_operands(over):
    """5000 rows sort: x 5000 x 128 bytes, the bank 4 x 32 x 128, ids 20,000 bytes, out 5000 x 64 bytes."""
    lib = _lib.lib()
    need = lib.vm_grouped_matmul_workspace(5000, 4)
    at = {"x": 1 << 24, "weight": 1 << 25, "ids": 1 << 26, "out": 1 << 27}
    size = {"x": 640000, "weight": 16384, "ids": 20000, "out": 320000}
    assert need > 0
    for where in (at[over], at[over] + size[over] // 32 * 16, at[over] - need // 32 * 16):
        assert _product(rows=5000, workspace=where, workspace_bytes=need, **at) == _lib.VM_EINVAL
        assert "the workspace overlaps an o" in _lib.last_error()


@pytest.mark.parametrize("over", ["base", "x", "a", "b", "scales", "ids", "out"])
def test_adapters_reject_a_workspace_over_their_operands(over):
    lib = _lib.lib()
    need = lib.vm_add_adapters_workspace(5000, 8, 4)
    at = {"base": 1 << 24, "x": 1 << 25, "a": 1 << 26, "b": 1 << 27, "scales": 1 << 28, "ids": 1 << 29, "out": 1 << 30}
    size = {"base": 320000, "x": 640000, "a": 4096, "b": 2048, "scales": 16, "ids": 20000, "out": 320000}
    assert need > 0
    for where in (at[over], at[over] + (size[over] - 1) // 16 * 16, at[over] - need // 32 * 16):
        assert _adapters(rows=5000, workspace=where, workspace_bytes=need, **at) == _lib.VM_EINVAL
        assert "the workspace overlaps an o" in _lib.last_error()
