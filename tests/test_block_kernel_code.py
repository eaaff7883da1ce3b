"""What the compiler made of the dense products and the block's norms, whose timings rely on it: registers, scratch, LDS, and
waits for loads, from one device-only compile to assembly of each source (no GPU needed)."""
import os
import re
import subprocess

import pytest

from veymoe import build

SOURCES = ("linear.hip", "linear_mx.hip", "block_norm.hip", "routing.hip")
_TEXT = {}


@pytest.fixture(scope="module")
def listings(tmp_path_factory):
    try:
        hipcc = build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc is not installed")
    if not _TEXT:
        path = tmp_path_factory.mktemp("listings")
        jobs = {}
        for name in SOURCES:
            out = path / f"{name}.s"
            cmd = [hipcc, *build.HIP_FLAGS, "--cuda-device-only", "-S", os.path.join(build.CSRC, name), "-o", str(out)]
            jobs[name] = subprocess.Popen(cmd, stdout=subprocess.DEVNULL, stderr=subprocess.PIPE, text=True), out
        for name, (proc, out) in jobs.items():
            _, err = proc.communicate()
            assert proc.returncode == 0, err[-2000:]
            _TEXT[name] = out.read_text()
    return _TEXT


def _kernels(text):
    return {name: {key: int(value) for key, value in re.findall(r"\.amdhsa_(\w+) (\d+)\n", body)}
            for name, body in re.findall(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", text, re.S)}


def test_no_kernel_takes_scratch(listings):
    for source, text in listings.items():
        kernels = _kernels(text)
        assert kernels
        assert {n: k["private_segment_fixed_size"] for n, k in kernels.items() if k["private_segment_fixed_size"]} == {}, source


def test_large_tiles_fit_a_cu(listings):
    """Two waves per SIMD: 256 registers a lane; four stages within the 160 KB of LDS, two blocks of the 128 x 128 tiles."""
    found = 0
    for source in ("linear.hip", "linear_mx.hip"):
        for name, k in _kernels(listings[source]).items():
            if "k_largeI" not in name:
                continue
            found += 1
            assert k["next_free_vgpr"] <= 256 and k["group_segment_fixed_size"] <= 160 * 1024, (name, k)
            if "ELi2ELi4ELi4ELi2EEE" in name:
                assert k["next_free_vgpr"] <= 128 and k["group_segment_fixed_size"] <= 80 * 1024, (name, k)
    assert found == 4 * 4 + 4 * 2


def test_large_tiles_wait_for_their_own_loads_only(listings):
    """Between the products no wait for all loads: the kernel leaves those of two steps on their way."""
    for source in ("linear.hip", "linear_mx.hip"):
        text = listings[source]
        for name in _kernels(text):
            if "k_largeI" not in name:
                continue
            start = text.index("\n" + name + ":")
            body = text[start:text.index("s_endpgm", start)]
            products = body[body.index("v_mfma"):body.rindex("v_mfma")]
            assert "vmcnt(0)" not in products, name
            assert re.search(r"vmcnt\(\d+\)", products), name
