"""ROUND_ONCE on the CPU: what takes the mode and what refuses it, and the code of its
kernels (the values are checked on the GPU, test_gpu_qkv_proj_i8_once.py)."""
import ctypes

from test_codegen import _asm, _counts
from test_int8_codegen import _mfmas
from test_int8_refusals import BUF, _qkv

ONCE = 3


def test_only_the_int8_projection_takes_it(h3):
    from h3hip import _lib
    lib = h3.lib()
    assert _lib.ROUND_ONCE == ONCE
    # Past the mode's check: refused for an address instead.
    odd = ctypes.c_void_p(4104)
    assert _qkv(h3, rounding=ONCE, q=odd) == _lib.EINVAL and "aligned" in h3.last_error()
    assert lib.h3hip_rope_table(BUF, BUF, BUF, 128, ONCE, 4, odd, None) == _lib.EINVAL
    assert "aligned" in h3.last_error()
    for rc in (lib.h3hip_qkv_proj(BUF, 128, BUF, 128, 64, BUF, BUF, 1e-6, BUF, 128, ONCE, 4, 128, 2,
                                  128, BUF, BUF, BUF, None),
               lib.h3hip_qk_norm_rope(BUF, BUF, 768, None, BUF, BUF, 1e-6, BUF, BUF, BUF, 128, ONCE,
                                      4, 128, 2, 128, BUF, BUF, None, None)):
        assert rc == _lib.EINVAL and "rounding" in h3.last_error()
    assert _qkv(h3, rounding=2) == _lib.EINVAL and "rounding" in h3.last_error()


def test_kernels_compiled_whole(tmp_path):
    """Two rotary widths of the eleven shapes that hold whole heads, nothing spilled; pairs
    of workgroups still share a CU."""
    asm = _asm(tmp_path, "proj_i8_once")
    spills, scratch = _counts(asm, "vgpr_spill_count"), _counts(asm, "private_segment_fixed_size")
    assert len(spills) == len(scratch) == 22
    assert max(spills) == 0 and max(scratch) == 0, (spills, scratch)
    assert _mfmas(asm) > 0
    lds, vgpr = _counts(asm, "group_segment_fixed_size"), _counts(asm, "vgpr_count")
    assert all(regs <= (256 if size <= 81920 else 512) for size, regs in zip(lds, vgpr))
