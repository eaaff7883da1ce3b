"""The argument checks of vm_select_experts, vm_block_norm and vm_linear, which reject bad calls before touching a device,
and the layouts of their argument structures (no GPU needed)."""
import ctypes
import os
import subprocess

import pytest

from veymoe import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "veymoe.h")
CONSTANTS = ("VM_SCORES_SOFTMAX", "VM_SCORES_SIGMOID", "VM_SELECT_MAX_EXPERTS", "VM_SELECT_MAX_GROUPS",
             "VM_SELECT_MAX_TOP_K", "VM_GATE_NONE", "VM_GATE_ROW", "VM_GATE_CHANNEL", "VM_GATE_VALUE",
             "VM_ACTIVATION_RELU", "VM_ACTIVATION_SILU", "VM_ACTIVATION_GELU", "VM_ACTIVATION_GELU_TANH",
             "VM_ACTIVATION_SIGMOID")


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"VmSelectArgs": _lib.VmSelectArgs, "VmBlockNormArgs": _lib.VmBlockNormArgs, "VmLinearArgs": _lib.VmLinearArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines += [f'printf("{c} %u\\n", (unsigned){c});' for c in CONSTANTS] + ["return 0; }"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    values = dict(line.rsplit(" ", 1) for line in out if line)
    for name, cls in structs.items():
        assert int(values[name]) == ctypes.sizeof(cls), name
        for field, _ in cls._fields_:
            assert int(values[f"{name}.{field}"]) == getattr(cls, field).offset, (name, field)
    for c in CONSTANTS:
        assert int(values[c]) == getattr(_lib, c), c


def _call(entry, cls, base, kw):
    a = cls()
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return getattr(_lib.lib(), entry)(ctypes.byref(a), None)


# two rows of 64 fp32 logits at 1 << 20
SELECT = {"logits": 1 << 20, "inds": 1 << 21, "weights": 1 << 22, "logits_stride": 64, "factor": 1.0, "rows": 2,
          "experts": 64, "groups": 1, "top_groups": 1, "group_top": 1, "top_k": 4, "logits_dtype": 1, "bias_dtype": 1,
          "weights_dtype": 1}


@pytest.mark.parametrize("fields,code,message", [
    ({"logits_dtype": 2}, _lib.VM_EINVAL, "dtypes"),
    ({"bias_dtype": 2}, _lib.VM_EINVAL, "dtypes"),
    ({"weights_dtype": 9}, _lib.VM_EINVAL, "dtypes"),
    ({"scores": 2}, _lib.VM_EINVAL, "scores"),
    ({"experts": 0}, _lib.VM_EUNSUPPORTED, "experts"),
    ({"experts": 1025}, _lib.VM_EUNSUPPORTED, "experts"),
    ({"groups": 0}, _lib.VM_EUNSUPPORTED, "groups"),
    ({"groups": 65, "experts": 130}, _lib.VM_EUNSUPPORTED, "groups"),
    ({"groups": 7}, _lib.VM_EUNSUPPORTED, "divide"),
    ({"top_groups": 0}, _lib.VM_EINVAL, "top_groups"),
    ({"groups": 4, "top_groups": 5}, _lib.VM_EINVAL, "top_groups"),
    ({"group_top": 0}, _lib.VM_EUNSUPPORTED, "group_top"),
    ({"group_top": 3}, _lib.VM_EUNSUPPORTED, "group_top"),
    ({"top_k": 0}, _lib.VM_EUNSUPPORTED, "top_k"),
    ({"top_k": 65, "experts": 100}, _lib.VM_EUNSUPPORTED, "top_k"),
    ({"top_k": 17, "groups": 4}, _lib.VM_EINVAL, "kept groups"),
    ({"rows": (1 << 25) + 1}, _lib.VM_EUNSUPPORTED, "rows"),
    ({"logits": None}, _lib.VM_EINVAL, "required"),
    ({"inds": None}, _lib.VM_EINVAL, "required"),
    ({"weights": None}, _lib.VM_EINVAL, "required"),
    ({"inds": (1 << 20) + 508}, _lib.VM_EINVAL, "overlap"),
    ({"weights": (1 << 20) - 28}, _lib.VM_EINVAL, "overlap"),
    ({"bias": (1 << 21) + 28}, _lib.VM_EINVAL, "overlap"),
    ({"weights": (1 << 21) + 28}, _lib.VM_EINVAL, "overlap"),
])
def test_select_rejects(fields, code, message):
    assert _call("vm_select_experts", _lib.VmSelectArgs, SELECT, fields) == code
    assert message in _lib.last_error()


# two bf16 rows of 64
NORM = {"x": 1 << 20, "residual": 1 << 21, "weight": 1 << 22, "out": 1 << 23, "sum_out": 1 << 24, "x_stride": 64,
        "residual_stride": 64, "gate_stride": 64, "out_stride": 64, "sum_stride": 64, "scale": 1.0, "residual_scale": 1.0,
        "eps": 1e-6, "rows": 2, "width": 64}
MX_OUT = {"out": None, "values": 1 << 25, "scales": 1 << 26}


@pytest.mark.parametrize("fields,code,message", [
    *[({f: 2}, _lib.VM_EINVAL, "dtypes") for f in ("act_dtype", "residual_dtype", "post_dtype", "gate_dtype", "weight_dtype")],
    ({"gate_kind": 4, "gate": 64}, _lib.VM_EINVAL, "gate_kind"),
    ({"gate_kind": 1}, _lib.VM_EINVAL, "go together"),
    ({"gate": 64}, _lib.VM_EINVAL, "go together"),
    ({"width": 0}, _lib.VM_EUNSUPPORTED, "width"),
    ({"width": 16385}, _lib.VM_EUNSUPPORTED, "width"),
    ({"rows": 1 << 24}, _lib.VM_EUNSUPPORTED, "rows"),
    ({"x": None}, _lib.VM_EINVAL, "required"),
    ({"residual": None}, _lib.VM_EINVAL, "required"),
    ({"out": None}, _lib.VM_EINVAL, "either out"),
    ({"values": 1 << 25, "scales": 1 << 26}, _lib.VM_EINVAL, "either out"),
    ({"weight": None}, _lib.VM_EINVAL, "one output"),
    ({"weight": None, **MX_OUT}, _lib.VM_EINVAL, "one output"),
    ({"weight": None, "out": None, "sum_out": None}, _lib.VM_EINVAL, "one output"),
    ({**MX_OUT, "scales": None}, _lib.VM_EINVAL, "both values and scales"),
    ({**MX_OUT, "width": 48}, _lib.VM_EINVAL, "multiple of 32"),
    ({**MX_OUT, "values": (1 << 25) + 4}, _lib.VM_EINVAL, "8-byte"),
    ({**MX_OUT, "scales": (1 << 25) + 100}, _lib.VM_EINVAL, "overlap"),
    ({"out_stride": 63}, _lib.VM_EINVAL, "strides of outputs"),
    ({"sum_stride": 63}, _lib.VM_EINVAL, "strides of outputs"),
    ({"out": (1 << 20) + 2}, _lib.VM_EINVAL, "overlap"),
    ({"out": 1 << 20, "out_stride": 72}, _lib.VM_EINVAL, "overlap"),
    ({"out": (1 << 22) + 126}, _lib.VM_EINVAL, "overlap"),
    ({"sum_out": (1 << 22) - 64}, _lib.VM_EINVAL, "overlap"),
    ({"sum_out": 1 << 23}, _lib.VM_EINVAL, "overlap"),
    ({"post_weight": (1 << 23) + 64}, _lib.VM_EINVAL, "overlap"),
    ({"gate": 1 << 23, "gate_kind": 3}, _lib.VM_EINVAL, "overlap"),
    ({"gate": (1 << 24) + 128, "gate_kind": 1}, _lib.VM_EINVAL, "overlap"),
    ({"gate": (1 << 24) + 128, "gate_kind": 2}, _lib.VM_EINVAL, "overlap"),
    # in place, but of another size of element
    ({"sum_out": 1 << 20, "residual_dtype": 1}, _lib.VM_EINVAL, "overlap"),
    ({"out": 1 << 21, "residual_dtype": 1}, _lib.VM_EINVAL, "overlap"),
    ({**MX_OUT, "values": 1 << 20}, _lib.VM_EINVAL, "MX rows overlap"),
    ({**MX_OUT, "scales": (1 << 24) + 64}, _lib.VM_EINVAL, "MX rows overlap"),
    ({**MX_OUT, "gate": 1 << 25, "gate_kind": 3}, _lib.VM_EINVAL, "MX rows overlap"),
])
def test_block_norm_rejects(fields, code, message):
    assert _call("vm_block_norm", _lib.VmBlockNormArgs, NORM, fields) == code
    assert message in _lib.last_error()


# two bf16 rows of 64 by a matrix of 32 rows
LINEAR = {"x": 1 << 20, "weight": 1 << 21, "out": 1 << 22, "x_stride": 64, "weight_stride": 64, "residual_stride": 32,
          "out_stride": 32, "rows": 2, "k": 64, "n": 32}
MX = {"format": _lib.VM_FORMAT_MX, "x_scales": 1 << 23, "weight_scales": 1 << 24, "x_scale_stride": 2, "weight_scale_stride": 2}


@pytest.mark.parametrize("fields,code,message", [
    ({"format": 2}, _lib.VM_EINVAL, "format"),
    ({"activation": 7}, _lib.VM_EINVAL, "activation"),
    *[({f: 2}, _lib.VM_EINVAL, "dtypes") for f in ("bias_dtype", "residual_dtype", "out_dtype")],
    ({"k": 0}, _lib.VM_EINVAL, "positive"),
    ({"n": 0}, _lib.VM_EINVAL, "positive"),
    ({"k": 60}, _lib.VM_EUNSUPPORTED, "multiple of 8"),
    ({**MX, "k": 48}, _lib.VM_EUNSUPPORTED, "multiple of 32"),
    ({"k": (1 << 24) + 8}, _lib.VM_EUNSUPPORTED, "2^24"),
    ({"n": (1 << 24) + 1}, _lib.VM_EUNSUPPORTED, "2^24"),
    ({"rows": (1 << 28) + 1}, _lib.VM_EUNSUPPORTED, "2^28"),
    ({"x": None}, _lib.VM_EINVAL, "required"),
    ({"weight": None}, _lib.VM_EINVAL, "required"),
    ({"out": None}, _lib.VM_EINVAL, "required"),
    ({**MX, "x_scales": None}, _lib.VM_EINVAL, "x_scales"),
    ({**MX, "weight_scales": None}, _lib.VM_EINVAL, "x_scales"),
    ({"x": (1 << 20) + 8}, _lib.VM_EINVAL, "16-byte"),
    ({"x_stride": 68}, _lib.VM_EINVAL, "16-byte"),
    ({"weight_stride": 68}, _lib.VM_EINVAL, "16-byte"),
    ({"out_stride": 31}, _lib.VM_EINVAL, "stride of out"),
    ({"rows": 1 << 28, "n": 1 << 24, "out_stride": 1 << 24}, _lib.VM_EUNSUPPORTED, "too large"),
    ({"out": (1 << 20) + 64}, _lib.VM_EINVAL, "overlaps an operand"),
    ({"out": (1 << 21) + 4094}, _lib.VM_EINVAL, "overlaps an operand"),
    ({"activation": 1, "out": (1 << 21) + 8190}, _lib.VM_EINVAL, "overlaps an operand"),
    ({"bias": (1 << 22) + 64}, _lib.VM_EINVAL, "overlaps an operand"),
    ({**MX, "out": 1 << 23}, _lib.VM_EINVAL, "overlaps an operand"),
    ({**MX, "out": (1 << 24) + 62}, _lib.VM_EINVAL, "overlaps an operand"),
    ({"residual": (1 << 22) + 2}, _lib.VM_EINVAL, "row for row"),
    ({"residual": 1 << 22, "residual_stride": 40}, _lib.VM_EINVAL, "row for row"),
    ({"residual": 1 << 22, "residual_dtype": 1}, _lib.VM_EINVAL, "row for row"),
])
def test_linear_rejects(fields, code, message):
    assert _call("vm_linear", _lib.VmLinearArgs, LINEAR, fields) == code
    assert message in _lib.last_error()


def test_calls_of_nothing():
    for entry, cls, base in (("vm_select_experts", _lib.VmSelectArgs, SELECT), ("vm_block_norm", _lib.VmBlockNormArgs, NORM),
                             ("vm_linear", _lib.VmLinearArgs, LINEAR)):
        assert _call(entry, cls, base, {"rows": 0}) == _lib.VM_OK
        assert getattr(_lib.lib(), entry)(None, None) == _lib.VM_EINVAL


def test_largest_legal_sizes_pass_the_checks_but_for_their_pointers():
    """Sizes at the documented limits are not refused for their size."""
    assert _call("vm_select_experts", _lib.VmSelectArgs, SELECT, {"rows": 1 << 25, "logits": None}) == _lib.VM_EINVAL
    assert "required" in _lib.last_error()
    wide = {"rows": 1 << 18, "n": 1 << 13, "out_stride": 1 << 13, "out": (1 << 20) + 64}
    assert _call("vm_linear", _lib.VmLinearArgs, LINEAR, wide) == _lib.VM_EINVAL
    assert "overlaps" in _lib.last_error()
