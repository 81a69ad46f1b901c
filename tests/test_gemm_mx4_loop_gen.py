"""The 4-bit projections' reduction loops (csrc/gen_gemm_mx4_loop.py ->
csrc/gemm_mx4_loop.inc), replayed on the CPU instruction by instruction.

The operands are the bf16 loops' (test_gemm_loop_gen.py says what its replay follows: which
step every LDS piece, operand register and accumulator holds, and the waits and barriers
between them). Here the scales join them: each product has to take, for either operand, the
byte of its own step and sub-step from a register that holds its own 16 rows' scales of that
pair of steps, landed behind a counted wait; a register is refilled only after the last
product that reads it; and the resources step on by one pair and are empty past the last.
Each of these mistakes is also planted once and must be found."""
import importlib.util
import os
import re

import pytest

from test_gemm_loop_gen import CSRC, Wrong, _drop, _span, check

spec = importlib.util.spec_from_file_location("gen_gemm_mx4_loop",
                                              os.path.join(CSRC, "gen_gemm_mx4_loop.py"))
G = importlib.util.module_from_spec(spec)
spec.loader.exec_module(G)
B = G.bf16

XS_STEP, WS_STEP = 1 << 20, 1 << 24       # bytes to the next pair's scales, told apart


def replay(g, lines, steps):
    labels = {ln[:-1]: i for i, ln in enumerate(lines) if ln.endswith(":")}
    pairs = (steps + 1) // 2
    s = {"%[steps]": steps, "%[pairs]": pairs, "%[m0w]": 0, "%[m0x]": 0, "m0": 0,
         "%[x_rec]": 1, "%[w_rec]": 1, "%[xs_rec]": 1, "%[ws_rec]": 1,
         "%[xs_step]": XS_STEP, "%[ws_step]": WS_STEP}
    scc = carry = False
    tile_pieces = {"w": g.na, "x": g.mb}
    piece, free_after = {}, {}
    vm, landed, lgkm, wait_barrier, barriers = [], 0, [], {}, 0
    regs, acc = {}, {}
    scales, in_use = {}, {}     # register -> (operand, block, pair, load number); reads left

    def val(t):
        return int(t, 0) if re.match(r"^-?(0x)?[0-9a-f]+$", t) else s.get(t, 0)

    pc = n = 0
    while pc < len(lines):
        n += 1
        check(n < 400000, "does not end")
        ln = lines[pc]
        pc += 1
        if ln.endswith(":"):
            continue
        op, _, rest = ln.partition(" ")
        a = [t.strip() for t in rest.split(",")]
        if op == "s_mov_b32":
            s[a[0]] = val(a[1])
        elif op in ("s_add_u32", "s_addc_u32"):
            total = val(a[1]) + val(a[2]) + (carry if op == "s_addc_u32" else 0)
            carry, s[a[0]] = total >= 1 << 32, total % (1 << 32)
        elif op in ("s_cmp_gt_u32", "s_cmp_lt_u32", "s_cmp_eq_u32"):
            x, y = val(a[0]), val(a[1])
            scc = {"gt": x > y, "lt": x < y, "eq": x == y}[op[6:8]]
        elif op == "s_cselect_b32":
            s[a[0]] = val(a[1]) if scc else val(a[2])
        elif op == "s_cbranch_scc1":
            pc = labels[a[0]] if scc else pc
        elif op == "s_branch":
            pc = labels[a[0]]
        elif op == "buffer_load_dwordx4":
            which = "x" if a[1] == B.XRS else "w"
            so, off = a[2].split()[0], int(re.search(r"offset:(\d+)", ln).group(1))
            rec = s["s66" if which == "x" else "s70"]
            step, k = divmod(s[so], B.ROW)
            check(k == 0)
            check(bool(rec) == (step < steps), "records", which, step)
            i = int(a[0][1:]) - (g.xv if which == "x" else g.wv)
            check(i % 4 * 1024 == off, "instruction offset", i, off)
            for w in range(4):
                at = (s["m0"] + off) // 1024 + tile_pieces[which] * w
                check(0 <= at * 1024 < g.lds)
                if at in free_after:
                    check(free_after[at] is not None and free_after[at] < barriers,
                          "refilled while read", which, step, at)
                piece[at] = (which, step if rec else None, tile_pieces[which] * w + i, len(vm))
                free_after[at] = None if rec else -1
            vm.append((which, step))
        elif op == "buffer_load_dword":
            reg = int(a[0][1:])
            which, lo, rec = ("x", "s80", "s82") if a[2] == G.XSRS else ("w", "s84", "s86")
            check(int(a[1][1:]) == g.sv and a[3].startswith("0 offen"), ln)
            pair, k = divmod(s[lo], XS_STEP if which == "x" else WS_STEP)
            check(k == 0, "base", s[lo])
            check(bool(s[rec]) == (pair < pairs), "scale records", which, pair)
            block, k = divmod(int(re.search(r"offset:(\d+)", ln).group(1)), 256)
            check(k == 0 and block < (g.na if which == "w" else g.mb))
            check(not in_use.get(reg), "scales refilled while needed", ln, in_use.get(reg))
            scales[reg] = (which, block, pair, len(vm))
            # Products that read it: both sub-steps of the pair's steps, over the other operand.
            uses = 2 * len([t for t in (2 * pair, 2 * pair + 1) if t < steps])
            in_use[reg] = uses * (g.mb if which == "w" else g.na)
            vm.append(("s", pair))
        elif op == "ds_read_b128":
            reg, (v, off) = _span(a[0]), a[1].split()
            v, off = int(v[1:]), int(off.split(":")[1])
            which = "w" if v < g.rb else "x"
            base, u = divmod(v - (g.ra if which == "w" else g.rb), 2)
            blocks = g.na if which == "w" else g.mb
            got, ats = set(), []
            for half in range(2):
                first = (off + 65536 * base) // 1024 + 2 * blocks * half
                for at in (first, first + 1):
                    check(at in piece, "read of an empty piece", ln)
                    kind, step, idx, num = piece[at]
                    check(kind == which and num in wait_barrier and wait_barrier[num] < barriers,
                          "read before its barrier", ln, step)
                    got.add((step, idx // 2 - blocks * half))
                    ats.append(at)
            check(len(got) == 1, "rows of different steps", ln, got)
            step, blk = got.pop()
            lgkm.append((reg, (which, step, u, blk), ats))
            for r in reg:
                regs[r] = "in flight"
        elif op == "s_waitcnt":
            m = re.search(r"vmcnt\((\d+)\)", ln)
            if m:
                while landed < len(vm) - int(m.group(1)):
                    wait_barrier[landed] = barriers
                    landed += 1
            m = re.search(r"lgkmcnt\((\d+)\)", ln)
            if m:
                while len(lgkm) > int(m.group(1)):
                    reg, what, ats = lgkm.pop(0)
                    for r in reg:
                        regs[r] = what
                    for at in ats:
                        free_after[at] = barriers
        elif op == "s_barrier":
            barriers += 1
        elif op == "v_mfma_scale_f32_16x16x128_f8f6f4":
            sb_reg, mods = a[5].split(" ", 1)
            mods += "," + ",".join(a[6:])
            sel = re.search(r"op_sel:\[(\d),(\d),0\] op_sel_hi:\[(\d),(\d),0\] cbsz:4 blgp:4", mods)
            check(sel, ln)
            lo_w, lo_x, hi_w, hi_x = map(int, sel.groups())
            c, ra, rb = _span(a[0]), _span(a[1]), _span(a[2])
            check(a[3] == a[0])
            A_, B_ = {regs.get(r) for r in ra}, {regs.get(r) for r in rb}
            check(len(A_) == 1 and len(B_) == 1 and not (A_ | B_) & {None, "in flight"}, "operand", ln)
            (kw, sa, ua, na), (kx, sb, ub, mb) = A_.pop(), B_.pop()
            check((kw, kx) == ("w", "x") and sa == sb and ua == ub, "operands of two steps", ln)
            check(c[0] == 4 * (g.mb * na + mb), "accumulator of another block", ln)
            for reg, which, block, byte in ((int(a[4][1:]), "w", na, 2 * hi_w + lo_w),
                                            (int(sb_reg[1:]), "x", mb, 2 * hi_x + lo_x)):
                check(reg in scales and scales[reg][3] in wait_barrier, "scales in flight", ln)
                check(scales[reg][:3] == (which, block, sa // 2), "another block's scales", ln)
                check(byte == 2 * (sa % 2) + ua, "byte of the scales", ln)
                in_use[reg] -= 1
            acc.setdefault(c[0], []).append((sa, ua))
        else:
            check(op in ("s_nop", "v_accvgpr_write_b32"), "unknown", ln)
    check(landed == len(vm) and not lgkm, "left in flight at the end")
    check(not any(in_use.values()), "scales not used up")
    check(sorted(acc) == list(range(0, 4 * g.na * g.mb, 4)))
    for c, seq in acc.items():
        check(seq == [(t, u) for t in range(steps) for u in range(2)], "sum", c, seq)


def _lines(name):
    g = G.Gen(name)
    return g, [ln.replace("%=", "") for ln in g.generate()]


def test_generated_file_is_current():
    assert open(G.OUT).read() == G.render()


@pytest.mark.parametrize("name", list(G.VARIANTS))
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 12, 13, 25])
def test_every_step_once_and_nothing_early(name, steps):
    g, lines = _lines(name)
    assert g.lds <= 163840 and g.n_vgpr <= 256
    replay(g, lines, steps)


@pytest.mark.parametrize("name", list(G.VARIANTS))
def test_registers_are_clobbered_or_inputs(name):
    """Every register the stream writes is declared: operands, scales and scalars."""
    g, lines = _lines(name)
    known = set(g.clobbers())
    for ln in lines:
        m = re.match(r"(?:ds_read_b128|buffer_load_dword) v\[?(\d+)(?::(\d+))?\]?,", ln)
        if m:
            for r in range(int(m.group(1)), int(m.group(2) or m.group(1)) + 1):
                assert f"v{r}" in known, ln
        m = re.match(r"s_\w+ s(\d+),", ln)
        if m and not ln.startswith("s_cmp"):
            assert f"s{m.group(1)}" in known, ln
    inputs = {at + i for _, at, k in g.inputs() for i in range(k)}
    assert not inputs & {int(r[1:]) for r in known if re.match(r"v\d", r)}


def _swap_bytes(lines):
    return [ln.replace("op_sel:[1,1,0]", "op_sel:[1,0,0]") for ln in lines]


PLANTED = {
    "a wait one load short": lambda g, ls: [
        re.sub(r"vmcnt\((\d+)\) lgkmcnt", lambda m: f"vmcnt({int(m.group(1)) + 1}) lgkmcnt", ln)
        for ln in ls],
    "a barrier missing": lambda g, ls: _drop(ls, "s_barrier", 2),
    "an operand read missing": lambda g, ls: _drop(ls, "ds_read_b128", 30),
    "a scale load missing": lambda g, ls: _drop(ls, "buffer_load_dword v", g.na + g.mb),
    "scales of one pair only": lambda g, ls: [ln for ln in ls if "%[ws_step]" not in ln],
    "scale records kept past the end": lambda g, ls: [ln for ln in ls
                                                      if ln != "s_cselect_b32 s82, s82, 0"],
    "the other byte of a scale": lambda g, ls: _swap_bytes(ls),
    "another set's scales": lambda g, ls: [
        ln.replace(f", v{g.sc} ", f", v{g.sc + 1} ").replace(f", v{g.sc},", f", v{g.sc + 1},")
        if "mfma" in ln else ln for ln in ls],
}


@pytest.mark.parametrize("name", list(G.VARIANTS))
@pytest.mark.parametrize("mistake", list(PLANTED))
def test_replay_finds_a_planted_mistake(name, mistake):
    g, lines = _lines(name)
    planted = PLANTED[mistake](g, lines)
    assert planted != lines
    with pytest.raises(Wrong):
        replay(g, planted, 13)
