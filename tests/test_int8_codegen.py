"""Code-generation properties of the int8 projections, checked on the CPU by compiling
them to gfx950 assembly (test_codegen.py has the bf16 kernels'): the reduction loops
carry all of their MFMAs, and nothing is spilled around them."""
import os
import re

from test_codegen import CSRC, _asm, _counts

FORMS = 6     # out-projection, plain QKV, and norm + RoPE in two roundings and two widths


def _mfmas(text):
    return sum(1 for ln in text.splitlines() if ln.strip(' "').startswith("v_mfma_i32_16x16x64_i8"))


def test_tile_kernels_compiled_whole(tmp_path):
    """Every shape in its forms: tiles narrower than a head only write token-major."""
    asm = _asm(tmp_path, "proj_i8_gemm")
    inc = open(os.path.join(CSRC, "gemm_i8_loop.inc")).read()
    forms, mfmas = 0, 0
    for part in re.split(r"(?=// \d+ channels x \d+ tokens)", inc)[1:]:
        n = FORMS if int(re.match(r"// (\d+)", part).group(1)) >= 128 else 1
        forms, mfmas = forms + n, mfmas + n * _mfmas(part)
    spills, scratch = _counts(asm, "vgpr_spill_count"), _counts(asm, "private_segment_fixed_size")
    assert len(spills) == len(scratch) == forms
    assert max(spills) == 0 and max(scratch) == 0, (spills, scratch)
    assert _mfmas(asm) == mfmas
    assert max(_counts(asm, "vgpr_count")) <= 512 and max(_counts(asm, "agpr_count")) <= 256


def test_pairs_share_a_cu(tmp_path):
    """Kernels with at most half the LDS leave a SIMD's registers for a second wave."""
    asm = _asm(tmp_path, "proj_i8_gemm")
    lds, vgpr = _counts(asm, "group_segment_fixed_size"), _counts(asm, "vgpr_count")
    assert len(lds) == len(vgpr) and min(lds) <= 81920
    for size, regs in zip(lds, vgpr):
        if size <= 81920:
            assert regs <= 256, (size, regs)


def test_quant_rows_spills_nothing(tmp_path):
    asm = _asm(tmp_path, "quant_rows")
    assert max(_counts(asm, "vgpr_spill_count")) == 0
    assert max(_counts(asm, "private_segment_fixed_size")) == 0
