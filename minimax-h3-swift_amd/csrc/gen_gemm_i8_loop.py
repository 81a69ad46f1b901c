#!/usr/bin/env python3
"""Writes gemm_i8_loop.inc: the reduction loops of the int8 projections
(proj_i8_kernel.h) as gfx950 inline assembly, one block per tile shape.

The stream is gen_gemm_loop.py's. A step's rows are 128 bytes there as here, 128
int8 values in place of 64 bf16 ones, and v_mfma_i32_16x16x64_i8 takes 16 bytes of
a row per lane as v_mfma_f32_16x16x32_bf16 does, in as many cycles, for twice the
products: loads, LDS layout, operand reads, waits and registers are the same, and so
is what they cost a step. Which k a lane's bytes stand for does not matter, because
both operands are read alike and the sum is exact.

Run `python3 gen_gemm_i8_loop.py` in this directory after editing either generator;
the generated file is committed, and tests/test_gemm_i8_loop_gen.py checks it is
current and replays it.
"""
from __future__ import annotations

import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)

import gen_gemm_loop as bf16  # noqa: E402

OUT = os.path.join(HERE, "gemm_i8_loop.inc")

# name (channels x tokens): (NA, MB, RW, RX). The shapes named p take at most half
# the LDS, so that two workgroups share a CU and one's waits are the other's work.
VARIANTS = {"256x256": (8, 8, 3, 2), "256x224": (8, 7, 3, 2), "256x192": (8, 6, 3, 2),
            "256x160": (8, 5, 3, 3), "256x128": (8, 4, 3, 3), "128x192": (4, 6, 4, 4),
            "128x160": (4, 5, 4, 4), "128x128": (4, 4, 5, 5),
            "128x128p": (4, 4, 2, 2), "128x64p": (4, 2, 3, 3), "128x32p": (4, 1, 4, 4),
            "64x64p": (2, 2, 5, 5), "32x64p": (1, 2, 6, 6), "32x32p": (1, 1, 8, 8)}


class Gen(bf16.Gen):
    VARIANTS = VARIANTS
    MFMA = "v_mfma_i32_16x16x64_i8"
    LABEL = "L_gemm_i8_"


def render():
    return bf16.render(Gen, "gen_gemm_i8_loop.py", "H3_GEMM_I8")


def main():
    text = render()
    if len(sys.argv) > 1 and sys.argv[1] == "--check":
        return 0 if os.path.exists(OUT) and open(OUT).read() == text else 1
    with open(OUT, "w") as f:
        f.write(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
