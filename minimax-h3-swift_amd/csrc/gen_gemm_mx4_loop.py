#!/usr/bin/env python3
"""Writes gemm_mx4_loop.inc: the reduction loops of the 4-bit projections
(proj_mx4_kernel.h) as gfx950 inline assembly, one block per tile shape.

The stream is gen_gemm_loop.py's. A step's rows are 128 bytes there as here, 256 4-bit
values in place of 64 bf16 ones: v_mfma_scale_f32_16x16x128_f8f6f4 on e2m1 operands takes
16 bytes of a row per lane as v_mfma_f32_16x16x32_bf16 does, in as many cycles, for four
times the products. A lane's 16 bytes are 32 consecutive values, one block with one
scale, and the product takes that scale as a byte of a register of the lane.

The scales come as the kernel reads them (quant_mx4.hip has their layout): a dword of a
lane holds its bytes for the two sub-steps of two steps, so that 16 rows' scales of a
pair of steps are one load of 256 consecutive bytes, straight into registers. The scales
of a pair are loaded `ahead` pairs before they are used, into one of ahead + 1 sets of
registers: at least as many steps as the rings look ahead, since a counted wait covers
everything issued before what it waits for. After the last pair the records are empty.

  v[..]        scale sets, A(set, na) and B(set, mb); then the lane's scale offset (input)
  s[80:88]     the scales' resources and the pair counter (clobbered)

Run `python3 gen_gemm_mx4_loop.py` in this directory after editing either generator;
the generated file is committed, and tests/test_gemm_mx4_loop_gen.py checks it is
current and replays it.
"""
from __future__ import annotations

import os
import sys
from math import lcm

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)

import gen_gemm_loop as bf16  # noqa: E402

OUT = os.path.join(HERE, "gemm_mx4_loop.inc")

# name (channels x tokens): (NA, MB, RW, RX). The shapes named p take at most half
# the LDS, so that two workgroups share a CU and one's waits are the other's work.
VARIANTS = {"256x256": (8, 8, 3, 2), "256x224": (8, 7, 3, 2), "256x192": (8, 6, 3, 2),
            "256x160": (8, 5, 3, 3), "256x128": (8, 4, 3, 3), "128x192": (4, 6, 4, 4),
            "128x160": (4, 5, 4, 4), "128x128": (4, 4, 5, 5),
            "128x128p": (4, 4, 2, 2), "128x64p": (4, 2, 3, 3), "128x32p": (4, 1, 4, 4),
            "64x64p": (2, 2, 5, 5), "32x64p": (1, 2, 6, 6), "32x32p": (1, 1, 8, 8)}

# Sets of scale registers by the deeper ring: what keeps the unrolled steps few.
SETS = {2: 2, 3: 3, 4: 4, 5: 5, 6: 3, 8: 4}

XSRS, WSRS, SPAIR = "s[80:83]", "s[84:87]", "s88"


class Gen(bf16.Gen):
    VARIANTS = VARIANTS
    MFMA = "v_mfma_scale_f32_16x16x128_f8f6f4"
    LABEL = "L_gemm_mx4_"

    def __init__(self, name):
        super().__init__(name)
        self.sets = SETS[max(self.rw, self.rx)]
        self.ahead = self.sets - 1
        self.unroll = lcm(self.rw, self.rx, 2 * self.sets)
        self.sc = self.n_vgpr
        self.sv = self.sc + self.sets * (self.na + self.mb)
        self.n_vgpr = self.sv + 1

    def scale(self, pair, which, k):
        return self.sc + (pair % self.sets) * (self.na + self.mb) + (k if which == "w" else self.na + k)

    def scale_load(self, slot, pair, which, k):
        self.issued.append(("s", pair))
        return [f"buffer_load_dword v{self.scale(slot, which, k)}, v{self.sv}, "
                f"{WSRS if which == 'w' else XSRS}, 0 offen offset:{256 * k}"]

    def next_pair(self):
        """Resources of the pair that follows; empty past the last."""
        return ["s_add_u32 s80, s80, %[xs_step]", "s_addc_u32 s81, s81, 0",
                "s_add_u32 s84, s84, %[ws_step]", "s_addc_u32 s85, s85, 0",
                f"s_add_u32 {SPAIR}, {SPAIR}, 1", f"s_cmp_lt_u32 {SPAIR}, %[pairs]",
                "s_cselect_b32 s82, s82, 0", "s_cselect_b32 s86, s86, 0"]

    def pair_calls(self, slot, pair):
        return ([lambda k=k: self.scale_load(slot, pair, "x", k) for k in range(self.mb)]
                + [lambda k=k: self.scale_load(slot, pair, "w", k) for k in range(self.na)]
                + [self.next_pair])

    def begin(self):
        for i, r in enumerate(("xs_lo", "xs_hi", "xs_rec")):
            self.emit(f"s_mov_b32 s{80 + i}, %[{r}]")
        for i, r in enumerate(("ws_lo", "ws_hi", "ws_rec")):
            self.emit(f"s_mov_b32 s{84 + i}, %[{r}]")
        self.emit("s_mov_b32 s83, 0x20000", "s_mov_b32 s87, 0x20000", f"s_mov_b32 {SPAIR}, 0")

    def lead(self):
        return max(super().lead(), 2 * self.ahead)

    def more_calls(self, t, step):
        if t % 2 or t // 2 + self.ahead < 0:
            return []
        return self.pair_calls(t // 2 + self.ahead, step // 2 + self.ahead)

    def needed(self, step):
        return super().needed(step) + ((("s", step // 2),) if step % 2 == 0 else ())

    def product(self, t, u, na, mb):
        sel = f"op_sel:[{u},{u},0] op_sel_hi:[{t % 2},{t % 2},0]"
        return (f"{super().product(t, u, na, mb)}, v{self.scale(t // 2, 'w', na)}, "
                f"v{self.scale(t // 2, 'x', mb)} {sel} cbsz:4 blgp:4")

    def inputs(self):
        return super().inputs() + [("SV", self.sv, 1)]

    def clobbers(self):
        return ([f"v{i}" for i in range(self.sc, self.sv)] + [f"s{i}" for i in range(80, 89)]
                + super().clobbers())


def render():
    return bf16.render(Gen, "gen_gemm_mx4_loop.py", "H3_GEMM_MX4")


def main():
    text = render()
    if len(sys.argv) > 1 and sys.argv[1] == "--check":
        return 0 if os.path.exists(OUT) and open(OUT).read() == text else 1
    with open(OUT, "w") as f:
        f.write(text)
    return 0


if __name__ == "__main__":
    sys.exit(main())
