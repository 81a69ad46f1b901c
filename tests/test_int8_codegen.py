"""Code-generation properties of the int8 projections, checked on the CPU by compiling
them to gfx950 assembly (test_codegen.py has the bf16 kernels'): the reduction loops
carry all of their MFMAs, and nothing is spilled around them."""
import os
import re

import pytest

from test_codegen import CSRC, _asm, _counts

FORMS = 6     # out-projection, plain QKV, and norm + RoPE in two roundings and two widths


def _mfmas(text):
    return sum(1 for ln in text.splitlines() if ln.strip(' "').startswith("v_mfma_i32_16x16x64_i8"))


def test_tile_kernels_compiled_whole(tmp_path):
    asm = _asm(tmp_path, "proj_i8_gemm")
    inc = open(os.path.join(CSRC, "gemm_i8_loop.inc")).read()
    shapes = len(re.findall(r"#define H3_GEMM_I8_LDS_", inc))
    spills, scratch = _counts(asm, "vgpr_spill_count"), _counts(asm, "private_segment_fixed_size")
    assert len(spills) == len(scratch) == shapes * FORMS
    assert max(spills) == 0 and max(scratch) == 0, (spills, scratch)
    assert _mfmas(asm) == FORMS * _mfmas(inc)
    assert max(_counts(asm, "vgpr_count")) <= 512 and max(_counts(asm, "agpr_count")) <= 256


@pytest.mark.parametrize("name", ["quant_rows", "proj_i8"])
def test_no_spills(tmp_path, name):
    asm = _asm(tmp_path, name)
    assert max(_counts(asm, "vgpr_spill_count")) == 0
    assert max(_counts(asm, "private_segment_fixed_size")) == 0
