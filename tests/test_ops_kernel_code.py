"""What the compiler made of the tiled products and adapters, whose timings rely on two blocks per CU: registers, scratch
and LDS, from one device-only compile to assembly of each source (no GPU needed)."""
import os
import re
import subprocess

import pytest

from veymoe import build

_FOUND = {}


def _kernels(source, tmp_path_factory):
    """{mangled name: {key: value}} of the kernels of csrc/``source``."""
    if not _FOUND:
        try:
            hipcc = build.hipcc()
        except RuntimeError:
            pytest.skip("hipcc is not installed")
        path = tmp_path_factory.mktemp("listings")
        jobs = {}
        for name in ("products.hip", "adapters.hip"):
            out = path / f"{name}.s"
            cmd = [hipcc, *build.HIP_FLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, name), "-o", str(out)]
            jobs[name] = subprocess.Popen(cmd, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True), out
        for name, (proc, out) in jobs.items():
            _, err = proc.communicate()
            assert proc.returncode == 0, err[-2000:]
            blocks = re.findall(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", out.read_text(), re.S)
            _FOUND[name] = {kernel: {key: int(value) for key, value in re.findall(r"\.amdhsa_(\w+) (\d+)\n", text)}
                            for kernel, text in blocks}
    return _FOUND[source]


def test_product_tiles_run_two_blocks_per_cu(tmp_path_factory):
    """Blocks of up to four waves: 256 registers a lane and half of the 160 KB of LDS.  Rows of whole chunks take no
    scratch."""
    tiles = {n: k for n, k in _kernels("products.hip", tmp_path_factory).items() if "k_tilesI" in n}
    assert len(tiles) == 6 * 4 * 2
    for name, k in tiles.items():
        assert k["next_free_vgpr"] <= 256 and k["group_segment_fixed_size"] <= 80 * 1024, (name, k)
        if name.split("EEEv")[0].endswith("Lb1"):
            assert k["private_segment_fixed_size"] == 0, (name, k)


def test_adapter_tiles_take_no_scratch(tmp_path_factory):
    """Ranks up to 64 run two blocks per CU at least; none spills."""
    tiles = {n: k for n, k in _kernels("adapters.hip", tmp_path_factory).items() if "k_adapter_tilesI" in n}
    assert tiles
    for name, k in tiles.items():
        assert k["private_segment_fixed_size"] == 0, (name, k)
        if "k_adapter_tilesILi8E" not in name:
            assert k["next_free_vgpr"] <= 256 and k["group_segment_fixed_size"] <= 80 * 1024, (name, k)


def test_no_product_instance_takes_scratch(tmp_path_factory):
    """Rows off whole chunks included."""
    kernels = _kernels("products.hip", tmp_path_factory)
    assert {n: k["private_segment_fixed_size"] for n, k in kernels.items() if k["private_segment_fixed_size"]} == {}
