"""Code-generation properties of the 4-bit projections, checked on the CPU by compiling them to
gfx950 assembly: the reduction loops carry all of their MFMAs, and nothing is spilled around
them."""
import os
import re

import pytest

from test_codegen import CSRC, _asm, _counts

LAUNCH = 120  # bytes of arguments: a launch of 128 and more takes the host longer
FORMS = 6     # out-projection, plain QKV, and norm + RoPE in two roundings and two widths


def _mfmas(text):
    return sum(1 for ln in text.splitlines()
               if ln.strip(' "').startswith("v_mfma_scale_f32_16x16x128_f8f6f4"))


def _check(asm):
    spills, scratch = _counts(asm, "vgpr_spill_count"), _counts(asm, "private_segment_fixed_size")
    assert max(spills) == 0 and max(scratch) == 0, (spills, scratch)
    # Kernels with at most half the LDS leave a SIMD's registers for a second wave.
    lds, vgpr = _counts(asm, "group_segment_fixed_size"), _counts(asm, "vgpr_count")
    assert len(lds) == len(vgpr) == len(spills) and min(lds) <= 81920
    assert max(_counts(asm, "kernarg_segment_size")) <= LAUNCH
    for size, regs in zip(lds, vgpr):
        assert regs <= (256 if size <= 81920 else 512), (size, regs)
    assert max(_counts(asm, "agpr_count")) <= 256
    return len(spills)


def test_tile_kernels_compiled_whole(tmp_path):
    """Every shape in its forms: tiles narrower than a head only write token-major."""
    asm = _asm(tmp_path, "proj_mx4_gemm")
    inc = open(os.path.join(CSRC, "gemm_mx4_loop.inc")).read()
    forms, mfmas = 0, 0
    for part in re.split(r"(?=// \d+ channels x \d+ tokens)", inc)[1:]:
        n = FORMS if int(re.match(r"// (\d+)", part).group(1)) >= 128 else 1
        forms, mfmas = forms + n, mfmas + n * _mfmas(part)
    assert _check(asm) == forms
    assert _mfmas(asm) == mfmas


def test_once_kernels_compiled_whole(tmp_path):
    """Two rotary widths of the shapes that hold whole heads."""
    asm = _asm(tmp_path, "proj_mx4_once")
    assert _check(asm) == 22 and _mfmas(asm) > 0


@pytest.mark.parametrize("source", ["quant_mx4", "few_mx4"])
def test_rows_spill_nothing(tmp_path, source):
    asm = _asm(tmp_path, source)
    assert max(_counts(asm, "vgpr_spill_count")) == 0
    assert max(_counts(asm, "private_segment_fixed_size")) == 0


def test_norms_spill_nothing(tmp_path):
    """And rows of one chunk a thread leave room for 24 waves a CU; rows of one segment, half of the
    kernels, launch with few arguments."""
    asm = _asm(tmp_path, "norm_residual")
    assert max(_counts(asm, "vgpr_spill_count")) == 0
    assert max(_counts(asm, "private_segment_fixed_size")) == 0
    vgpr = _counts(asm, "vgpr_count")
    assert len(vgpr) == 20 and sorted(vgpr)[9] <= 80 and max(vgpr) <= 128, vgpr
    assert sorted(_counts(asm, "kernarg_segment_size"))[9] <= LAUNCH
