"""The forms that the tests of linear's forms are meant to reach are those that it chooses, and every one is among them (from the
host's choice, compiled alone; no GPU needed)."""
import os
import subprocess

import pytest

from linear_forms import FORMS
from veymoe import build

NAMES = ["few", "16", "32", "32x64", "64", "64deep", "128", "128x320", "256", "256x320"]
MAIN = r"""
#include <stdio.h>
#include "%s/vm_linear_form.h"
int main(void) {
  unsigned mx, rows, n, k, pairs, large;
  while (scanf("%%u %%u %%u %%u %%u %%u", &mx, &rows, &n, &k, &pairs, &large) == 6) {
    const vm::LinearForm c = mx ? vm::choose_form<true>(rows, n, k, pairs, large) : vm::choose_form<false>(rows, n, 2 * k, pairs, large);
    printf("%%d %%llu %%u %%d %%d\n", c.form, (unsigned long long)c.blocks, c.threads, c.alone, c.fits());
  }
  for (int f = 0; f < vm::kForms; ++f)
    printf("%%d %%u %%u %%u %%u %%u %%u\n", f, vm::kTileForms<false>[f].rows, vm::kTileForms<false>[f].matrix,
           vm::kTileForms<false>[f].places, vm::kTileForms<true>[f].rows, vm::kTileForms<true>[f].matrix, vm::kTileForms<true>[f].places);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    path = tmp_path_factory.mktemp("forms")
    (path / "forms.cpp").write_text(MAIN % build.CSRC)
    subprocess.run(["g++", "-std=c++17", "-O1", str(path / "forms.cpp"), "-o", str(path / "forms")], check=True)
    return str(path / "forms")


def _choices(program, calls):
    """(name, blocks, threads, alone, fits) of (mx, rows, n, k, pairs, large) and the tables."""
    text = "\n".join(" ".join(str(int(v)) for v in c) for c in calls) + "\n."
    lines = subprocess.run([program], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
    rows = [[int(v) for v in line.split()] for line in lines if line]
    return [(NAMES[r[0] + 1], *r[1:3], bool(r[3]), bool(r[4])) for r in rows[:len(calls)]], rows[len(calls):]


def test_calls_reach_their_forms(program):
    calls = [(mx, rows, n // 2 if pairs else n, k, pairs, not mx or k % 128 == 0)
             for _, _, mx, rows, k, n in FORMS for pairs in (False, True)]
    chosen, _ = _choices(program, calls)
    assert [c[0] for c in chosen] == [f[0] for f in FORMS for _ in range(2)]
    assert [c[3] for c in chosen] == [f[1] for f in FORMS for _ in range(2)]


def test_every_form_is_reached(program):
    _, tables = _choices(program, [])
    for mx in (False, True):
        there = {"few"} | {NAMES[r[0] + 1] for r in tables if r[6 if mx else 3] > 0}
        assert {f[0] for f in FORMS if f[2] == mx} == there
        for name in ("16", "32"):     # of which a lone tile has an instance of its own
            assert {f[1] for f in FORMS if f[2] == mx and f[0] == name} == {True, False}


def test_grids_cover_their_calls(program):
    """Whole tiles over rows and matrix rows, none more, whatever the sizes."""
    calls = [(mx, rows, n, k, pairs, large) for mx in (0, 1) for rows in (1, 4, 5, 16, 17, 63, 200, 1000, 4097, 70000, 1 << 28)
             for n in (1, 2, 15, 64, 333, 2560, 40001, 1 << 24) for k in (32, 96, 1024, 8192, 1 << 24) for pairs in (0, 1)
             for large in (0, 1)]
    chosen, tables = _choices(program, calls)
    for (mx, rows, n, _, pairs, large), (name, blocks, threads, alone, fits) in zip(calls, chosen):
        matrix = n * (2 if pairs else 1)
        if rows <= 4:
            assert name == "few" and blocks == -(-matrix // 4)
            continue
        t = tables[NAMES.index(name) - 1][4 if mx else 1:][:3]
        assert t[2] > 0 and blocks == -(-rows // t[0]) * -(-matrix // t[1]) and alone == (blocks <= 256)
        assert large or name not in ("128", "128x320", "256", "256x320")
        assert fits == (blocks * threads < 1 << 32)


def test_the_header_stands_alone():
    text = open(os.path.join(build.CSRC, "vm_linear_form.h")).read()
    assert "#include <stdint.h>" in text and text.count("#include") == 1
