"""The rule by which the norms' kernels are launched (csrc/norm_rule.h, compiled here with g++),
against the registers that the kernels compile to: of few rows no more workgroups than fit a CU,
and never more than a second round of them."""
import os
import re
import shutil
import subprocess

import pytest

from test_codegen import CSRC, _asm

HARNESS = r"""
#include "norm_rule.h"
#include <cstdio>
#include <initializer_list>
using namespace h3hip;
int main() {
  for (int form = 0; form < 32; form++) {
    const int simd = norm_waves_simd(form & 1 ? 2 : 1, form & 2, form & 4, form & 8, form & 16);
    std::printf("%d", simd);
    for (int rows : {1, 300, 4095, 4096, 31885})
      for (int waves = 1; waves <= 16; waves++)
        std::printf(" %d", norm_workers_cu(waves, rows, simd));
    std::printf("\n");
  }
}
"""
ROWS = (1, 300, 4095, 4096, 31885)


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    d = tmp_path_factory.mktemp("norm")
    (d / "t.cpp").write_text(HARNESS)
    subprocess.run([gxx, "-O1", "-std=c++17", f"-I{CSRC}", str(d / "t.cpp"), "-o", str(d / "t")],
                   check=True)
    out = subprocess.run([str(d / "t")], check=True, capture_output=True, text=True).stdout
    return [[int(v) for v in ln.split()] for ln in out.splitlines()]


def _forms(asm):
    """(form of the harness, VGPRs) of each compiled kernel."""
    for c, flags, vgpr in re.findall(
            r"\.symbol:\s+\S*norm_residual_kernelILi(\d)E((?:Lb[01]E){4})\S*\.kd\s.*?\.vgpr_count:\s+(\d+)",
            asm, re.S):
        bits = [int(b) for b in re.findall(r"Lb([01])E", flags)]
        yield (int(c) - 1) + sum(b << (i + 1) for i, b in enumerate(bits)), int(vgpr)


def test_workgroups_fit_the_registers(rule, tmp_path):
    forms = dict(_forms(_asm(tmp_path, "norm_residual")))
    assert len(forms) == 20
    for form, vgpr in forms.items():
        room = 4 * (512 // (-(-vgpr // 8) * 8))           # waves a CU, registers in eights
        assert rule[form][0] * 4 <= room, (form, vgpr)
        for i, rows in enumerate(ROWS):
            for waves in range(1, 17):
                n = rule[form][1 + 16 * i + waves - 1]
                assert n >= 1
                if rows < 4096:
                    assert n * waves <= max(room, waves), (form, vgpr, rows, waves)
                assert n <= max(1, 2 * (room // waves)), (form, vgpr, rows, waves)


def test_more_rows_never_fewer_workgroups(rule):
    for line in rule:
        for waves in range(16):
            n = [line[1 + 16 * i + waves] for i in range(len(ROWS))]
            assert n == sorted(n)
