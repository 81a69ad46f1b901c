#!/usr/bin/env python3
"""Headline benchmark: block-sparse attention TFLOP/s over active tiles (and
the fraction of the bf16 MFMA peak) at the 1344x768x5s shape, plus ms/layer.

One step = one DiT layer's hot path at config 3 (S = 31,885 -> 32,000,
40 heads x 128, local-window mask, 7,854 active 128x128 tiles per head):
  1. the fused prologue: Q/K RMSNorm + 3D RoPE + head-major relayout of Q and
     K, read from a token-major fused qkv buffer;
  2. block-sparse attention over the plan's tiles, V read in place from the
     fused buffer (a strided view, as the reference's SDPA receives it),
     written token-major ([S, heads*128], what the out-projection consumes).
The tile plan is built once per shape (timed separately, not per layer).
Inputs are synthetic and already resident in HBM when the timed region starts.

    python bench.py [--gpus 1] [--steps 20] [--warmup 10] [--no-cpu-baseline] [--no-extras]
"""
from __future__ import annotations

import argparse
import json
import math
import os
import sys
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(ROOT, "minimax-h3-swift_amd"))

METRIC = "block-sparse attn TFLOP/s (active tiles) + % MFMA peak at 31k tokens; ms/layer"
PEAK_BF16_TFLOPS = 2500.0     # MI355X dense bf16 MFMA, spec sheet
PEAK_HBM_GBPS = 8000.0        # MI355X HBM3E, spec sheet
FLOP_PER_TILE_HEAD = 4 * 128 ** 3   # QK^T and PV over one 128x128 tile, head_dim 128
C_HIDDEN = 5120               # the benchmark configs' model width (input of the QKV projection)


def read_profile_value(name: str, key: str):
    """A `key: value` figure from a committed rocprofv3 summary, if any."""
    path = os.path.join(ROOT, "profiles", name)
    if not os.path.exists(path):
        return None
    for line in open(path):
        if line.startswith(key + ":"):
            return float(line.split(":", 1)[1])
    return None


def read_traffic(name: str):
    """HBM bytes per launch from a committed rocprofv3 --pmc summary, if any."""
    return read_profile_value(name, "traffic_bytes_per_launch")


def useful_tile_flops(plan_rows, seq_len: int, heads: int, tile: int = 128, d: int = 128):
    """FLOPs of the active tiles without their padding: 4 * d * (query rows <
    seq_len) * (key columns < seq_len) summed over the tiles, times heads."""
    row_ptr, col_idx = plan_rows
    total = 0
    for qt in range(len(row_ptr) - 1):
        rows = min(tile, seq_len - qt * tile)
        cols = sum(min(tile, seq_len - int(kt) * tile) for kt in col_idx[row_ptr[qt]:row_ptr[qt + 1]])
        total += rows * cols
    return 4 * d * total * heads


def interleaved_medians(fns: dict, reps: int = 12, warmup: int = 2) -> dict:
    """Median per-call milliseconds of each callable, the calls interleaved in
    alternating order (A B C, C B A, A B C, ...), each bracketed by HIP events on
    the stream it launches on (torch's current stream) -- the interleaved-median
    discipline of the reference's BenchmarkSupport.swift:10-30."""
    import numpy as np
    import torch
    names = list(fns)
    for _ in range(warmup):
        for n in names:
            fns[n]()
    ev = {n: [] for n in names}
    for r in range(reps):
        for n in (names if r % 2 == 0 else names[::-1]):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            fns[n]()
            b.record()
            ev[n].append((a, b))
    torch.cuda.synchronize()
    return {n: float(np.median([a.elapsed_time(b) for a, b in ev[n]])) for n in names}


def host_cpu():
    """CPU model, logical CPUs and the threads OpenMP would use on this host."""
    model = "unknown"
    try:
        for line in open("/proc/cpuinfo"):
            if line.startswith("model name"):
                model = line.split(":", 1)[1].strip()
                break
    except OSError:
        pass
    try:
        avail = len(os.sched_getaffinity(0))
    except AttributeError:
        avail = os.cpu_count() or 1
    return model, os.cpu_count() or 1, avail, os.environ.get("OMP_NUM_THREADS")


def cpu_baseline(shape, plan_rows, seconds: float = 12.0):
    """The reference path on the host CPU: the oracle's restatement of
    AxialReference.attend (fp32, additive -1e30 mask over all S keys) on a
    bounded sample of config 3 -- one head, rows spread over every q-tile --
    scaled to active-tile TFLOP/s so it reads in the metric's unit."""
    import numpy as np
    sys.path.insert(0, os.path.join(ROOT, "oracle"))
    import oracle as O
    row_ptr, col_idx = plan_rows
    n = len(row_ptr) - 1
    bm = np.zeros((n, n), dtype=np.uint8)
    for i in range(n):
        bm[i, col_idx[row_ptr[i]:row_ptr[i + 1]]] = 1
    S, D = shape.seq_len, 128
    rng = np.random.default_rng(0)
    k = rng.standard_normal((S, D), dtype=np.float32)
    v = rng.standard_normal((S, D), dtype=np.float32)
    model, nproc, avail, omp_env = host_cpu()
    # Every host CPU this process may run on, at most the 16 that the GPU box
    # allots to one GPU.
    threads = min(16, avail)

    rows = np.arange(S, dtype=np.int32)
    q = rng.standard_normal((S, D), dtype=np.float32)
    row_len = np.diff(row_ptr).astype(np.int64)
    head_flops = int(row_len[rows // 128].sum()) * 128 * D * 4   # active-tile FLOPs, one head

    def one_head():
        t0 = time.perf_counter()
        O.attend_rows(q, rows, k, v, 1.0 / math.sqrt(D), bm, tile=128, threads=threads)
        return time.perf_counter() - t0

    first = one_head()
    n_heads = int(max(1, min(shape.heads - 1, math.ceil(seconds / max(first, 1e-3)) - 1)))
    dt = first + sum(one_head() for _ in range(n_heads))
    n_heads += 1

    # Config 1 in full (all 4 heads, every row) through the same restatement.
    from h3hip import configs as C
    c1 = C.CFG1
    bm1 = O.tile_bitmap(O.Rule(**c1.oracle_rule_kwargs()))
    q1 = rng.standard_normal((c1.heads, c1.seq_len, D), dtype=np.float32)
    k1 = rng.standard_normal((c1.heads, c1.seq_len, D), dtype=np.float32)
    v1 = rng.standard_normal((c1.heads, c1.seq_len, D), dtype=np.float32)
    t0 = time.perf_counter()
    O.attend_masked(q1, k1, v1, 1.0 / math.sqrt(D), bm1, tile=128, threads=threads)
    dt1 = time.perf_counter() - t0
    flops1 = int(bm1.sum()) * c1.heads * 4 * 128 ** 2 * D

    # The prologue on the host, in full at config 5's size (Q and K, every
    # token and head), through the oracle's restatement in reference rounding.
    inner = shape.heads * D
    pos = O.positions_grid(shape.prefix_len, shape.frames, shape.height, shape.width)
    ax, inv = O.rope_pairs_axes(1.0e4, 32, 48, 48)
    gam = O.uniform_bf16((D,), 3, 0.9, 1.1)
    t_pro = 0.0
    for seed in (1, 2):
        x = O.randn_bf16((S, inner), seed)
        t0 = time.perf_counter()
        O.qk_norm_rope(x, inner, S, shape.seq_pad, shape.heads, D, gam, 1e-6, pos, ax, inv,
                       128, threads=threads)
        t_pro += time.perf_counter() - t0
        del x
    pro_bytes = 2 * S * inner * 2 + 2 * shape.seq_pad * inner * 2 + S * 12 + 2 * D * 2
    return {
        "value": round(n_heads * head_flops / dt / 1e12, 6),
        "unit": "TFLOP/s",
        "cores": threads,
        "cpu_model": model,
        "nproc": nproc,
        "cpus_available": avail,
        "omp_num_threads_env": omp_env,
        "kind": "port",
        "sample": (f"oracle dense-masked attention (AxialReference.attend restated in C, "
                   f"OpenMP, fp32, every query row scored against all {S} keys) on {n_heads} of "
                   f"the {shape.heads} heads of config 3 in {dt:.1f} s; value = active-tile "
                   f"FLOPs of those heads / time; a full layer would take "
                   f"{dt / n_heads * shape.heads:.0f} s"),
        "cfg1_full": {"seconds": round(dt1, 3),
                      "tflops_active": round(flops1 / dt1 / 1e12, 6),
                      "sample": "config 1 (4 heads x 4,096 rows, band rule) in full"},
        "prologue_cfg5_full": {"seconds": round(t_pro, 3),
                               "gbps": round(pro_bytes / t_pro / 1e9, 2),
                               "sample": ("Q and K of config 5 (31,885 tokens x 40 heads) in "
                                          "full, reference rounding")},
    }


def profile_only(args, env) -> int:
    """One kernel in isolation, for rocprofv3 counter runs."""
    import torch
    from h3hip import ops
    dev, H, D, S, S_pad = env["dev"], env["H"], env["D"], env["S"], env["S_pad"]
    if args.only == "copy":
        src = torch.empty(1 << 29, dtype=torch.int16, device=dev).fill_(1)
        dst = torch.empty_like(src)
        for _ in range(args.warmup + args.steps):
            dst.copy_(src)
        torch.cuda.synchronize()
        print(f"copy: {args.steps} x {src.numel() * 2} bytes read and written")
        return 0
    if args.only == "anchor":
        fns, notes, plan, keep = sdpa_anchor_fns(dev)
        names = [n for n in ("h3hip_bsattn_fwd", "torch_flash_aotriton") if n in fns]
        for _ in range(args.warmup + args.steps):
            for n in names:
                fns[n]()
        torch.cuda.synchronize()
        print(f"anchor: {args.steps} launches each of {', '.join(names)} at [1, 40, 18176, 128]"
              + (f"; {notes}" if notes else ""))
        plan.close()
        return 0
    if args.only == "mfma_ceiling":
        cus = torch.cuda.get_device_properties(dev).multi_processor_count
        fns, _, keep = mfma_ceiling_fns(dev, cus)
        for _ in range(args.warmup + args.steps):
            fns["mfma32_random"]()
        torch.cuda.synchronize()
        print(f"mfma_ceiling: {args.steps} launches of the 32x32x16 stream on random operands")
        return 0
    if args.only == "issue":
        cus = torch.cuda.get_device_properties(dev).multi_processor_count
        res = issue_probe(dev, cus)
        print("issue: " + "; ".join(f"{k} ({v['what']}) {v['cycles_per_iter']} cycles, "
                                     f"MFMA busy {v['mfma_busy']}" for k, v in res.items()))
        return 0
    if args.only == "qkv":
        x, w = qkv_inputs(env)
        vh = torch.empty_like(env["qh"])
        table = ops.rope_table(env["pos"], env["ax"], env["inv"])
        for _ in range(args.warmup + args.steps):
            ops.qkv_proj(x, w, env["gq"], env["gk"], table, heads=H, eps=env["C"].QK_EPS,
                         seq_pad=S_pad, out=(env["qh"], env["kh"], vh))
        torch.cuda.synchronize()
        print(f"qkv: {args.steps} launches, x [{S}, {C_HIDDEN}] x W^T -> Q, K, V [{H}, {S_pad}, {D}]")
        return 0
    if args.only == "gemms":
        # This library's plain and fused QKV projections, hipBLASLt's QKV GEMM
        # (torch.mm), this library's and hipBLASLt's out-projection, in turn.
        x, w = qkv_inputs(env)
        w_out = (torch.randn((C_HIDDEN, H * D), generator=env["g"], device=dev) * 0.02).to(torch.bfloat16)
        vh = torch.empty_like(env["qh"])
        qkv = torch.empty((S, 3 * H * D), dtype=torch.bfloat16, device=dev)
        y = torch.empty((S, C_HIDDEN), dtype=torch.bfloat16, device=dev)
        att = x[:, :H * D]
        table = ops.rope_table(env["pos"], env["ax"], env["inv"])
        out = (env["qh"], env["kh"], vh)
        for _ in range(args.warmup + args.steps):
            ops.qkv_proj(x, w, heads=H, seq_pad=S_pad, out=out)
            torch.mm(x, w.t(), out=qkv)
            ops.qkv_proj(x, w, env["gq"], env["gk"], table, heads=H, eps=env["C"].QK_EPS,
                         seq_pad=S_pad, out=out)
            ops.out_proj(att, w_out, out=y)
            torch.mm(att, w_out.t(), out=y)
        torch.cuda.synchronize()
        print(f"gemms: {args.steps} rounds of plain QKV, hipBLASLt QKV, fused QKV, out-projection, "
              f"hipBLASLt out-projection at config 3")
        return 0
    if args.only == "attention":
        env["prologue"]()
        for _ in range(args.warmup + args.steps):
            env["attention"]()
        torch.cuda.synchronize()
        print(f"attention: {args.steps} launches at {env['shape'].name}")
        return 0
    g, inner = env["g"], H * D
    q_in = torch.randn((S, inner), generator=g, device=dev).to(torch.bfloat16)
    k_in = torch.randn((S, inner), generator=g, device=dev).to(torch.bfloat16)
    for _ in range(args.warmup + args.steps):
        ops.qk_norm_rope(q_in, k_in, env["gq"], env["gk"], env["pos"], env["ax"], env["inv"],
                         heads=H, eps=1e-6, seq_pad=S_pad, out=(env["qh"], env["kh"], None))
    torch.cuda.synchronize()
    print(f"prologue: {args.steps} launches, Q and K [{S}, {inner}] -> [{H}, {S_pad}, {D}]")
    return 0


def probe_lib():
    """libch3probe.so: same-run hardware ceilings (MFMA stream, HBM streams),
    built beside libch3hip.so and not part of the attention path."""
    import ctypes
    path = os.path.join(ROOT, "minimax-h3-swift_amd", "libch3probe.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is not built; run __graft_entry__.build()")
    L = ctypes.CDLL(path)
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    L.h3probe_mfma_operand_bytes.restype, L.h3probe_mfma_operand_bytes.argtypes = i64, [i32]
    L.h3probe_mfma_flops.restype, L.h3probe_mfma_flops.argtypes = ctypes.c_double, [i32, i32]
    L.h3probe_mfma.restype = ctypes.c_int
    L.h3probe_mfma.argtypes = [i32, vp, i32, i32, vp, vp]
    L.h3probe_stream.restype = ctypes.c_int
    L.h3probe_stream.argtypes = [i32, vp, vp, i64, i32, i32, vp, vp]
    L.h3probe_relayout.restype = ctypes.c_int
    L.h3probe_relayout.argtypes = [i32, vp, vp, i32, i32, i32, vp]
    L.h3probe_issue_operand_bytes.restype, L.h3probe_issue_operand_bytes.argtypes = i64, [i32]
    L.h3probe_issue.restype = ctypes.c_int
    L.h3probe_issue.argtypes = [i32, vp, i32, i32, vp, vp]
    return L


def _stream_ptr():
    import torch
    return ctypes_ptr(torch.cuda.current_stream().cuda_stream)


def ctypes_ptr(x):
    import ctypes
    return ctypes.c_void_p(int(x))


def mfma_ceiling_fns(dev, cus: int, iters: int = 2000):
    """Launchers of the sustained-MFMA probe (one workgroup of 8 waves per CU):
    v_mfma_f32_32x32x16_bf16 (the attention kernel's shape) and
    v_mfma_f32_16x16x32_bf16 (the projection's), on N(0,1) bf16 operands and on
    zeros. Returns ({name: fn}, FLOPs per launch)."""
    import torch
    P = probe_lib()
    n = P.h3probe_mfma_operand_bytes(cus) // 2
    g = torch.Generator(device=dev)
    g.manual_seed(99)
    rnd = torch.randn(n, generator=g, device=dev).to(torch.bfloat16)
    zero = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    sink = torch.empty(cus * 512, dtype=torch.float32, device=dev)

    def mk(shape, ops):
        def fn():
            rc = P.h3probe_mfma(shape, ctypes_ptr(ops.data_ptr()), cus, iters,
                                ctypes_ptr(sink.data_ptr()), _stream_ptr())
            assert rc == 0, f"h3probe_mfma returned {rc}"
        return fn
    fns = {"mfma32_random": mk(0, rnd), "mfma32_zero": mk(0, zero),
           "mfma16_random": mk(1, rnd), "mfma32_agpr_acc_random": mk(2, rnd)}
    return fns, P.h3probe_mfma_flops(cus, iters), (rnd, zero, sink)


ISSUE_MIXES = {0: "4 mfma32", 1: "4 mfma32 + 4 x (fma, max3, exp)",
               2: "mix 1 + 2 v_dot2c_f32_bf16", 3: "mix 1 + 4 v_add_f32",
               4: "mix 1 + 1 v_mfma_f32_4x4x4bf16_1k"}


def issue_probe(dev, cus: int, iters: int = 4000) -> dict:
    """Shader-clock cycles per iteration of each issue mix (probes/ceilings.hip,
    issue_mix: four v_mfma_f32_32x32x16_bf16 with the mix's instructions after
    them, 8 waves per CU on random operands). Per workgroup the slowest of its
    waves gives the iteration time of a SIMD running two of them; the median
    over workgroups is reported, with the matrix cores' busy fraction
    (8 MFMAs x 32 cycles per iteration per SIMD)."""
    import numpy as np
    import torch
    P = probe_lib()
    g = torch.Generator(device=dev)
    g.manual_seed(17)
    ops = torch.randn(P.h3probe_issue_operand_bytes(cus) // 2, generator=g,
                      device=dev).to(torch.bfloat16)
    cyc = torch.zeros(cus * 8, dtype=torch.int64, device=dev)
    out = {}
    for mix, label in ISSUE_MIXES.items():
        for _ in range(2):   # the first launch warms up
            rc = P.h3probe_issue(mix, ctypes_ptr(ops.data_ptr()), cus, iters,
                                 ctypes_ptr(cyc.data_ptr()), _stream_ptr())
            assert rc == 0, f"h3probe_issue returned {rc}"
        torch.cuda.synchronize()
        per_wg = cyc.view(cus, 8).max(dim=1).values.cpu().numpy() / iters
        c = float(np.median(per_wg))
        out[f"mix{mix}"] = {"what": label, "cycles_per_iter": round(c, 1),
                            "mfma_busy": round(8 * 32 / c, 4)}
    return out


RELAYOUT_VARIANTS = {0: "tokens-fastest 8x5x512", 1: "tokens-fastest 2x5x256",
                     2: "tokens-fastest 4x4x256", 3: "heads-fastest 4x4x256",
                     4: "2x2 blocks 4x5x512", 8: "tokens-fastest 16x5x512",
                     5: "tokens-fastest 8x5x512, default cache policy",
                     6: "tokens-fastest 4x4x256, default cache policy",
                     7: "tokens-fastest 16x5x512, default cache policy",
                     9: "tokens-fastest 32x5x512, default cache policy"}


def ceilings_extra(args, dev, cus: int, read_bytes: int, write_bytes: int, relayout=None):
    """The chip's sustained MFMA rate per shape (power-limited at real data),
    the best HBM read-only, write-only and read+write streams of the prologue's
    byte counts, swept over grid size and per-thread unroll, and the best of
    several thread mappings of the prologue's layout change alone (token-major
    Q|K -> head-major, no arithmetic; relayout = (rows, rows_pad, heads)), in
    this run."""
    import torch
    fns, flops, keep = mfma_ceiling_fns(dev, cus)
    med = interleaved_medians(fns, reps=6, warmup=2)
    res = {"timing": "medians of interleaved calls",
           "mfma_probe": ("one workgroup of 8 waves per CU, 4 independent accumulator chains "
                          "per wave, operands in registers, 2,000 iterations")}
    for name, ms in med.items():
        res[name + "_tflops"] = round(flops / (ms * 1e-3) / 1e12, 1)
        res[name + "_peak_frac"] = round(flops / (ms * 1e-3) / 1e12 / PEAK_BF16_TFLOPS, 4)
    del keep
    res["issue_probe"] = issue_probe(dev, cus)
    P = probe_lib()
    nbytes = max(read_bytes, write_bytes)
    src = torch.empty(nbytes // 2, dtype=torch.bfloat16, device=dev).fill_(1.0)
    dst = torch.empty_like(src)
    sink = torch.empty(1 << 16, dtype=torch.int32, device=dev)
    sweep = [(b, u) for b in (1024, 2048, 4096, 8192) for u in (2, 4, 8)]

    def mk(kind, nb, blocks, unroll):
        def fn():
            rc = P.h3probe_stream(kind, ctypes_ptr(src.data_ptr()), ctypes_ptr(dst.data_ptr()),
                                  nb, blocks, unroll, ctypes_ptr(sink.data_ptr()), _stream_ptr())
            assert rc == 0, f"h3probe_stream returned {rc}"
        return fn
    for kind, label, nb, moved in ((0, "read", read_bytes, read_bytes),
                                   (1, "write", write_bytes, write_bytes),
                                   (2, "copy", read_bytes, 2 * read_bytes)):
        m = interleaved_medians({f"{b}x{u}": mk(kind, nb, b, u) for b, u in sweep},
                                reps=8, warmup=2)
        best = min(m, key=m.get)
        res[f"{label}_stream"] = {"bytes": moved, "best_ms": round(m[best], 4),
                                  "best_gbps": round(moved / (m[best] * 1e-3) / 1e9, 1),
                                  "best_grid_x_unroll": best,
                                  "worst_gbps": round(moved / (max(m.values()) * 1e-3) / 1e9, 1)}
    if relayout is not None:
        rows, rows_pad, heads = relayout
        rin = src[:rows * heads * 128]
        rout = dst[:heads * rows_pad * 128]

        def mkr(v):
            def fn():
                rc = P.h3probe_relayout(v, ctypes_ptr(rin.data_ptr()), ctypes_ptr(rout.data_ptr()),
                                        rows, rows_pad, heads, _stream_ptr())
                assert rc == 0, f"h3probe_relayout returned {rc}"
            return fn
        m = interleaved_medians({RELAYOUT_VARIANTS[v]: mkr(v) for v in RELAYOUT_VARIANTS},
                                reps=8, warmup=2)
        moved = (rows + rows_pad) * heads * 256
        best = min(m, key=m.get)
        res["relayout_stream"] = {"bytes": moved, "best_ms": round(m[best], 4),
                                  "best_gbps": round(moved / (m[best] * 1e-3) / 1e9, 1),
                                  "best_mapping": best,
                                  "by_mapping_gbps": {k: round(moved / (v * 1e-3) / 1e9, 1)
                                                      for k, v in m.items()}}
    rd, wr = res["read_stream"], res["write_stream"]
    # Reads then writes of the prologue's bytes, each at its own best rate: a
    # kernel that overlapped them perfectly could at best reach the copy's rate.
    res["read_then_write_ms"] = round(rd["best_ms"] + wr["best_ms"], 4)
    res["read_then_write_gbps"] = round((read_bytes + write_bytes)
                                        / ((rd["best_ms"] + wr["best_ms"]) * 1e-3) / 1e9, 1)
    del src, dst, sink
    return res


def sdpa_anchor_inputs(dev, heads: int = 40, seq: int = 18176):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(4321)
    q, k, v = (torch.randn((1, heads, seq, 128), generator=g, device=dev).to(torch.bfloat16)
               for _ in range(3))
    return q, k, v


def sdpa_anchor_fns(dev, heads: int = 40, seq: int = 18176):
    """Dense attention at config 4's padded shape ([1, 40, 18,176, 128] bf16,
    no mask, every tile active) through torch's fused SDPA kernels -- the
    flash backend (AOTriton on this ROCm build, and CK where the build has it)
    and the memory-efficient backend -- beside this library's kernel on a
    dense plan of the same length. The math backend is never allowed, so a
    backend that cannot run raises instead of falling back."""
    import torch
    import h3hip
    from h3hip import ops
    from torch.nn.attention import SDPBackend, sdpa_kernel
    q, k, v = sdpa_anchor_inputs(dev, heads, seq)
    out = torch.empty_like(q)
    plan = h3hip.TilePlan(h3hip.MaskRule.dense(seq), heads=heads)
    scale = 1.0 / math.sqrt(128)
    fns, notes = {}, {}

    def ours():
        ops.bsattn_fwd(plan, q[0], k[0], v[0], scale, out=out[0])
    fns["h3hip_bsattn_fwd"] = ours

    def sdpa_with(backend, lib=None):
        def fn():
            if lib is not None:
                torch.backends.cuda.preferred_rocm_fa_library(lib)
            with sdpa_kernel([backend]):
                torch.nn.functional.scaled_dot_product_attention(q, k, v, scale=scale)
        return fn
    cands = [("torch_flash_aotriton", SDPBackend.FLASH_ATTENTION, "aotriton"),
             ("torch_flash_ck", SDPBackend.FLASH_ATTENTION, "ck"),
             ("torch_mem_efficient", SDPBackend.EFFICIENT_ATTENTION, None)]
    for name, backend, lib in cands:
        fn = sdpa_with(backend, lib)
        try:
            fn()
            torch.cuda.synchronize()
            fns[name] = fn
        except Exception as e:  # a backend this build or GPU does not have
            notes[name] = f"did not run: {type(e).__name__}: {str(e).splitlines()[0][:160]}"
    try:
        torch.backends.cuda.preferred_rocm_fa_library("default")
    except Exception:
        pass
    return fns, notes, plan, (q, k, v, out)


def sdpa_anchor_extra(args, dev):
    """Same-run anchor for the attention kernel's roofline: dense attention at
    config 4's padded shape through torch's fused SDPA backends, interleaved
    with h3hip_bsattn_fwd on a dense plan, plus a max-abs difference of each
    output from ours."""
    import torch
    fns, notes, plan, keep = sdpa_anchor_fns(dev)
    q, k, v, out = keep
    heads, seq = q.shape[1], q.shape[2]
    flops = 4.0 * heads * seq * seq * 128
    med = interleaved_medians(fns, reps=max(10, args.steps // 2), warmup=2)
    res = {"timing": "medians of interleaved calls",
           "shape": f"[1, {heads}, {seq}, 128] bf16, no mask (all {plan.nnz} tiles per head)",
           "tflop_per_call": round(flops / 1e12, 4)}
    fns["h3hip_bsattn_fwd"]()
    ref = out.float()
    for name, ms in med.items():
        entry = {"ms": round(ms, 4), "tflops": round(flops / (ms * 1e-3) / 1e12, 1),
                 "peak_frac": round(flops / (ms * 1e-3) / 1e12 / PEAK_BF16_TFLOPS, 4)}
        if name != "h3hip_bsattn_fwd":
            from torch.nn.attention import sdpa_kernel, SDPBackend
            be = (SDPBackend.EFFICIENT_ATTENTION if "efficient" in name
                  else SDPBackend.FLASH_ATTENTION)
            if name == "torch_flash_ck":
                torch.backends.cuda.preferred_rocm_fa_library("ck")
            with sdpa_kernel([be]):
                o = torch.nn.functional.scaled_dot_product_attention(
                    q, k, v, scale=1.0 / math.sqrt(128))
            torch.backends.cuda.preferred_rocm_fa_library("default")
            entry["max_abs_diff_vs_h3hip"] = round(float((o.float() - ref).abs().max()), 5)
            del o
        res[name] = entry
    res.update(notes)
    plan.close()
    del keep, ref
    return res


def qkv_inputs(env):
    """Config 3's projection operands: x [S, 5120] N(0,1), qkvWeight
    [3*heads*128, 5120] N(0, 0.02^2), bf16."""
    import torch
    g, dev, S, inner = env["g"], env["dev"], env["S"], env["H"] * env["D"]
    x = torch.randn((S, C_HIDDEN), generator=g, device=dev).to(torch.bfloat16)
    w = (torch.randn((3 * inner, C_HIDDEN), generator=g, device=dev) * 0.02).to(torch.bfloat16)
    return x, w


def qkv_projection_extra(args, env):
    """The fused projection (GEMM + Q/K norm/RoPE + head-major relayout in one
    kernel) against hipBLASLt's GEMM (torch.mm) followed by the prologue kernel,
    at config 3. Both leave the layer's attention inputs ready (the unfused V
    stays token-major in the qkv buffer, read in place)."""
    import numpy as np
    import torch
    from h3hip import ops
    H, S, S_pad, inner = env["H"], env["S"], env["S_pad"], env["H"] * env["D"]
    x, w = qkv_inputs(env)
    qh, kh = env["qh"], env["kh"]
    vh = torch.empty_like(qh)
    qkv_tmp = torch.empty((S, 3 * inner), dtype=torch.bfloat16, device=env["dev"])
    tables = (env["gq"], env["gk"], env["pos"], env["ax"], env["inv"])
    # The rotation table is built once per render (prepareRender), not per layer.
    table = ops.rope_table(env["pos"], env["ax"], env["inv"])

    def fused():
        r = ops.qkv_proj(x, w, env["gq"], env["gk"], table, heads=H, eps=env["C"].QK_EPS,
                         seq_pad=S_pad, out=(qh, kh, vh))
        assert r is not None

    def gemm():
        torch.mm(x, w.t(), out=qkv_tmp)

    def prologue():
        ops.qk_norm_rope(qkv_tmp[:, :inner], qkv_tmp[:, inner:2 * inner], *tables, heads=H,
                         eps=env["C"].QK_EPS, seq_pad=S_pad, out=(qh, kh, None))

    med = interleaved_medians({"fused": fused, "gemm": gemm, "prologue": prologue},
                              reps=max(12, args.steps))
    t = [med["fused"], med["gemm"], med["prologue"]]
    flops = 2.0 * S * C_HIDDEN * 3 * inner
    tf = lambda ms: round(flops / (ms * 1e-3) / 1e12, 1)
    return {"timing": "medians of interleaved calls", "fused_ms": round(t[0], 4),
            "fused_tflops": tf(t[0]),
            "fused_mfma_peak_frac": round(flops / (t[0] * 1e-3) / 1e12 / PEAK_BF16_TFLOPS, 4),
            "hipblaslt_gemm_ms": round(t[1], 4), "hipblaslt_gemm_tflops": tf(t[1]),
            "prologue_after_gemm_ms": round(t[2], 4),
            "unfused_ms": round(t[1] + t[2], 4),
            "gemm_tflop": round(flops / 1e12, 4)}


def attention_layer_extra(args, env):
    """AttentionLayer.callAsFunction (DiTBlock.swift:336-359) at config 3, end to
    end: QKV projection + Q/K norm/RoPE, block-sparse attention, out-projection.
    Three paths: every kernel this library's (fused projection, attention,
    h3hip_out_proj); the fused projection with hipBLASLt's out-projection
    (torch.mm); and hipBLASLt's GEMMs with the prologue kernel between them
    (V then read in place from the token-major qkv). The out-projection alone
    is timed both ways beside them. Then the first path in turn with the same layer on
    int8 projections (weights rounded before, activations in the timed call)."""
    import numpy as np
    import torch
    from h3hip import ops
    H, D, S, S_pad = env["H"], env["D"], env["S"], env["S_pad"]
    inner = H * D
    x, w = qkv_inputs(env)
    g, dev = env["g"], env["dev"]
    w_out = (torch.randn((C_HIDDEN, inner), generator=g, device=dev) * 0.02).to(torch.bfloat16)
    plan, scale = env["plan"], env["scale"]
    qh, kh = env["qh"], env["kh"]
    vh = torch.empty_like(qh)
    qkv = torch.empty((S, 3 * inner), dtype=torch.bfloat16, device=dev)
    att = torch.empty((S, inner), dtype=torch.bfloat16, device=dev)
    att_view = att.view(S, H, D).transpose(0, 1)
    v_view = qkv[:, 2 * inner:].view(S, H, D).transpose(0, 1)
    y = torch.empty((S, C_HIDDEN), dtype=torch.bfloat16, device=dev)
    table = ops.rope_table(env["pos"], env["ax"], env["inv"])
    eps = env["C"].QK_EPS

    def all_h3hip_path():
        ops.qkv_proj(x, w, env["gq"], env["gk"], table, heads=H, eps=eps, seq_pad=S_pad,
                     out=(qh, kh, vh))
        ops.bsattn_fwd_strided(plan, qh, kh, vh, scale, out=att_view)
        ops.out_proj(att, w_out, out=y)

    def fused_path():
        ops.qkv_proj(x, w, env["gq"], env["gk"], table, heads=H, eps=eps, seq_pad=S_pad,
                     out=(qh, kh, vh))
        ops.bsattn_fwd_strided(plan, qh, kh, vh, scale, out=att_view)
        torch.mm(att, w_out.t(), out=y)

    def unfused_path():
        torch.mm(x, w.t(), out=qkv)
        ops.qk_norm_rope(qkv[:, :inner], qkv[:, inner:2 * inner], env["gq"], env["gk"],
                         env["pos"], env["ax"], env["inv"], heads=H, eps=eps, seq_pad=S_pad,
                         out=(qh, kh, None))
        ops.bsattn_fwd_strided(plan, qh, kh, v_view, scale, out=att_view)
        torch.mm(att, w_out.t(), out=y)

    def out_h3hip():
        ops.out_proj(att, w_out, out=y)

    def out_hipblaslt():
        torch.mm(att, w_out.t(), out=y)

    med = interleaved_medians({"all_h3hip": all_h3hip_path, "fused_qkv": fused_path,
                               "hipblaslt_qkv": unfused_path, "out_proj_h3hip": out_h3hip,
                               "out_proj_hipblaslt": out_hipblaslt},
                              reps=max(12, args.steps))
    res = {"timing": "medians of interleaved calls",
           "paths": {"all_h3hip": "fused QKV projection + attention + out-projection, all this "
                                  "library's kernels",
                     "fused_qkv": "fused QKV projection + attention + hipBLASLt out-projection",
                     "hipblaslt_qkv": "hipBLASLt QKV GEMM + prologue + attention + hipBLASLt "
                                      "out-projection"}}
    for name, ms in med.items():
        res[name + "_ms"] = round(ms, 4)
    out_flops = 2.0 * S * inner * C_HIDDEN
    res["out_proj_h3hip_tflops"] = round(out_flops / (med["out_proj_h3hip"] * 1e-3) / 1e12, 1)
    res["out_proj_hipblaslt_tflops"] = round(out_flops / (med["out_proj_hipblaslt"] * 1e-3) / 1e12, 1)
    flops = (2.0 * S * C_HIDDEN * 3 * inner + plan.nnz * H * FLOP_PER_TILE_HEAD + out_flops)
    res["layer_tflop"] = round(flops / 1e12, 4)
    best = min(res["all_h3hip_ms"], res["fused_qkv_ms"], res["hipblaslt_qkv_ms"])
    res["best_tflops"] = round(flops / (best * 1e-3) / 1e12, 1)

    w8, w8_out = ops.quant_rows(w), ops.quant_rows(w_out)
    x8, att8 = (tuple(torch.empty_like(t) for t in ops.quant_rows(a)) for a in (x, att))
    y8 = torch.empty_like(y)

    def int8_path():
        ops.quant_rows(x, out=x8)
        ops.qkv_proj_i8(*x8, *w8, env["gq"], env["gk"], table, heads=H, eps=eps, seq_pad=S_pad,
                        out=(qh, kh, vh))
        ops.bsattn_fwd_strided(plan, qh, kh, vh, scale, out=att_view)
        ops.quant_rows(att, out=att8)
        ops.proj_i8(*att8, *w8_out, out=y8)

    med = interleaved_medians({"bf16": all_h3hip_path, "int8": int8_path},
                              reps=max(12, args.steps))
    rel = float((y8.double() - y.double()).norm() / y.double().norm())
    res["int8_projections"] = {"timing": "medians of interleaved calls",
                               "int8_ms": round(med["int8"], 4), "bf16_ms": round(med["bf16"], 4),
                               "rel_rms_vs_bf16": round(rel, 5)}
    return res


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--warmup", type=int, default=10)
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-extras", action="store_true")
    ap.add_argument("--only", choices=("attention", "prologue", "copy", "qkv", "gemms", "anchor",
                                       "mfma_ceiling", "issue"),
                    help="profiling mode: run one kernel --steps times at config 3 (prologue: "
                         "config 5, Q and K only; copy: a plain 1 GiB device copy for counter "
                         "calibration; qkv: the fused QKV projection; gemms: the projections and "
                         "hipBLASLt's GEMMs of the same shapes in turn; anchor: this library's "
                         "attention and torch's flash SDPA alternately, dense, at config 4's "
                         "padded shape; mfma_ceiling: the sustained 32x32x16 MFMA stream; "
                         "issue: the MFMA/VALU issue-mix probe, printed per mix) and print "
                         "nothing but a one-line summary")
    args = ap.parse_args()
    world = int(os.environ.get("WORLD_SIZE", "1"))
    if args.gpus != 1 or world != 1:
        print(f"bench.py measures one GPU only (asked for --gpus {args.gpus}, WORLD_SIZE "
              f"{world}): the path shards by heads with no communication inside attention, "
              f"so N GPUs run N independent copies of this measurement.", file=sys.stderr)
        return 2

    import numpy as np
    import torch

    import h3hip
    from h3hip import configs as C, ops

    dev = torch.device("cuda:0")
    shape = C.CFG3
    S, S_pad, H, D = shape.seq_len, shape.seq_pad, shape.heads, C.HEAD_DIM
    inner = H * D

    # ---- plan (once per shape) --------------------------------------------
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    plan = h3hip.TilePlan(shape.mask_rule(), heads=H)
    tile_build_ms = (time.perf_counter() - t0) * 1e3
    t0 = time.perf_counter()
    plan.close()
    plan = h3hip.TilePlan(shape.mask_rule(), heads=H)
    tile_build_ms = min(tile_build_ms, (time.perf_counter() - t0) * 1e3)
    attn_flops = plan.nnz * H * FLOP_PER_TILE_HEAD
    attn_useful_flops = useful_tile_flops(plan.tiles(), S, H)
    clk = read_profile_value("bsattn_fwd_cfg3_clock.txt", "effective_clock_ghz")

    # ---- synthetic inputs, resident in HBM ----------------------------------
    g = torch.Generator(device=dev)
    g.manual_seed(1234)
    qkv = torch.randn((S, 3 * inner), generator=g, device=dev).to(torch.bfloat16)
    gq = (torch.rand(D, generator=g, device=dev) * 0.2 + 0.9).to(torch.bfloat16)
    gk = (torch.rand(D, generator=g, device=dev) * 0.2 + 0.9).to(torch.bfloat16)
    pos = torch.from_numpy(ops.positions_grid(shape.prefix_len, shape.frames, shape.height,
                                              shape.width)).to(dev)
    ax_np, inv_np = ops.rope_pairs_axes(C.ROPE_THETA, C.ROPE_DIMS)
    ax, inv = torch.from_numpy(ax_np).to(dev), torch.from_numpy(inv_np).to(dev)
    qh = torch.empty((H, S_pad, D), dtype=torch.bfloat16, device=dev)
    kh = torch.empty_like(qh)
    out = torch.empty((S, inner), dtype=torch.bfloat16, device=dev)
    # [H, S, D] views: V in place in the fused projection output, and the
    # token-major output.
    v_view = qkv[:, 2 * inner:].view(S, H, D).transpose(0, 1)
    out_view = out.view(S, H, D).transpose(0, 1)
    scale = 1.0 / math.sqrt(D)

    def prologue():
        r = ops.qk_norm_rope(qkv[:, :inner], qkv[:, inner:2 * inner], gq, gk, pos, ax, inv,
                             heads=H, eps=C.QK_EPS, seq_pad=S_pad, out=(qh, kh, None))
        assert r is not None

    def attention():
        r = ops.bsattn_fwd_strided(plan, qh, kh, v_view, scale, out=out_view)
        assert r is not None

    if args.only:
        return profile_only(args, locals())

    for _ in range(args.warmup):
        prologue()
        attention()
    torch.cuda.synchronize()

    ev = [[torch.cuda.Event(enable_timing=True) for _ in range(3)] for _ in range(args.steps)]
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for i in range(args.steps):
        ev[i][0].record()
        prologue()
        ev[i][1].record()
        attention()
        ev[i][2].record()
    torch.cuda.synchronize()
    wall_ms = (time.perf_counter() - t0) * 1e3
    # Per-launch durations from events on the stream the kernels run on
    # (torch's current stream); the roofline uses the average launch.
    pro_ms = float(np.mean([e[0].elapsed_time(e[1]) for e in ev]))
    attn_ms = float(np.mean([e[1].elapsed_time(e[2]) for e in ev]))
    attn_median_ms = float(np.median([e[1].elapsed_time(e[2]) for e in ev]))
    ms_per_step = wall_ms / args.steps
    attn_tflops = attn_flops / (attn_ms * 1e-3) / 1e12
    pro_bytes = 2 * S * inner * 2 + 2 * S_pad * inner * 2 + S * 12 + 2 * D * 2
    pro_gbps = pro_bytes / (pro_ms * 1e-3) / 1e9
    assert torch.isfinite(out.float()).all()

    result = {
        "metric": METRIC,
        "value": round(attn_tflops, 3),
        "unit": "TFLOP/s",
        "n_gpus": 1,
        "steps": args.steps,
        "warmup": args.warmup,
        "ms_per_step": round(ms_per_step, 4),
        "higher_is_better": True,
        "scaling": "weak",
        "vs_baseline": None,
        "dtype": "bf16",
        "data": "synthetic: seeded bf16 N(0,1) fused qkv [S, 3*5120], gamma U(0.9,1.1), integer (t,h,w) grid positions",
        "config": {
            "workload": shape.name,
            "seq_len": S, "seq_pad": S_pad, "heads": H, "head_dim": D,
            "video_grid": [shape.frames, shape.height, shape.width],
            "text_tokens": shape.text, "audio_tokens": shape.audio,
            "mask_rule": "local window: prefix rows/cols dense, +-1 latent frame, 3x3 spatial tiles of 8x8",
            "active_tiles_per_head": plan.nnz, "tile_density": round(plan.density, 5),
            "step": "prologue(Q,K norm+RoPE+relayout) + block-sparse attention (V in place in the fused qkv, token-major out)",
        },
        "attn_ms": round(attn_ms, 4),
        "attn_ms_median": round(attn_median_ms, 4),
        "attn_tflop_per_launch": round(attn_flops / 1e12, 4),
        "attn_tflops_active": round(attn_tflops, 3),
        "attn_mfma_peak_frac": round(attn_tflops / PEAK_BF16_TFLOPS, 4),
        # The same rate against the dense bf16 peak at a clock NOT measured in
        # this run: the committed profile's cycles per XCD (GRBM_GUI_ACTIVE)
        # over its unprofiled duration, from an earlier run and possibly another
        # box. Context only; the roofline fraction is against the spec peak.
        "attn_profiled_clock_ghz": clk,
        "attn_profiled_clock_source": "profiles/bsattn_fwd_cfg3_clock.txt (an earlier run)",
        "attn_mfma_peak_frac_at_profiled_clock": (
            round(attn_tflops / (PEAK_BF16_TFLOPS * clk / 2.4), 4) if clk else None),
        # Without the padding rows and columns inside the active tiles.
        "attn_useful_tflop_per_launch": round(attn_useful_flops / 1e12, 4),
        "attn_useful_tflops": round(attn_useful_flops / (attn_ms * 1e-3) / 1e12, 3),
        "prologue_qk_ms": round(pro_ms, 4),
        "prologue_qk_gbps": round(pro_gbps, 1),
        "ms_per_layer": round(pro_ms + attn_ms, 4),
        "tile_build_ms_once_per_shape": round(tile_build_ms, 2),
        "roofline": {
            "bound": "mfma",
            "achieved": round(attn_tflops, 3),
            "peak": PEAK_BF16_TFLOPS,
            "unit": "TFLOP/s",
            "frac": round(attn_tflops / PEAK_BF16_TFLOPS, 4),
            "traffic": read_traffic("bsattn_fwd_cfg3_traffic.txt"),
        },
    }

    if not args.no_extras:
        extras = {}
        # Config 5: the prologue alone (Q, K only), fed by the hidden->Q,K setup GEMM.
        hidden = torch.randn((S_pad, 5120), generator=g, device=dev).to(torch.bfloat16)
        wq = (torch.randn((5120, inner), generator=g, device=dev) * 0.02).to(torch.bfloat16)
        q_in = (hidden @ wq)[:S]
        k_in = (hidden @ ((torch.randn((5120, inner), generator=g, device=dev) * 0.02)
                          .to(torch.bfloat16)))[:S]
        del hidden, wq
        # The same bytes moved by a plain device copy and by the pure token ->
        # head-major relayout of Q and K (h3hip_head_major, no arithmetic): the
        # ceilings the prologue's layout change runs against, in the same run.
        qk_in = torch.empty((S, 2 * inner), dtype=torch.bfloat16, device=dev)
        qk_in[:, :inner].copy_(q_in)
        qk_in[:, inner:].copy_(k_in)
        qk_hm = torch.empty((2 * H, S_pad, D), dtype=torch.bfloat16, device=dev)
        copy_src = torch.empty(2 * S_pad * inner, dtype=torch.bfloat16, device=dev).fill_(1.0)
        copy_dst = torch.empty_like(copy_src)
        med = interleaved_medians({
            "prologue": lambda: ops.qk_norm_rope(q_in, k_in, gq, gk, pos, ax, inv, heads=H,
                                                 eps=C.QK_EPS, seq_pad=S_pad,
                                                 out=(qh, kh, None)),
            "relayout": lambda: ops.head_major(qk_in, heads=2 * H, seq_pad=S_pad, out=qk_hm),
            "copy": lambda: copy_dst.copy_(copy_src),
        }, reps=max(12, args.steps))
        b5 = 2 * S * inner * 2 + 2 * S_pad * inner * 2 + S * 12 + 2 * D * 2
        b_rel = 2 * S * inner * 2 + 2 * S_pad * inner * 2
        b_copy = 2 * copy_src.numel() * 2
        gbps = lambda b, ms: round(b / (ms * 1e-3) / 1e9, 1)
        p5 = med["prologue"]
        extras["cfg5_prologue_qk"] = {
            "timing": "medians of interleaved calls",
            "ms": round(p5, 4), "bytes": b5, "gbps": gbps(b5, p5),
            "hbm_peak_frac": round(b5 / (p5 * 1e-3) / 1e9 / PEAK_HBM_GBPS, 4),
            "relayout_ceiling_ms": round(med["relayout"], 4),
            "relayout_ceiling_gbps": gbps(b_rel, med["relayout"]),
            "copy_ceiling_ms": round(med["copy"], 4),
            "copy_ceiling_gbps": gbps(b_copy, med["copy"]),
            "frac_of_relayout_ceiling": round(gbps(b5, p5) / gbps(b_rel, med["relayout"]), 4),
            "traffic": read_traffic("qk_norm_rope_cfg5_traffic.txt"),
        }
        result["prologue_relayout_ceiling_gbps"] = extras["cfg5_prologue_qk"]["relayout_ceiling_gbps"]
        result["prologue_copy_ceiling_gbps"] = extras["cfg5_prologue_qk"]["copy_ceiling_gbps"]
        del q_in, k_in, qk_in, qk_hm, copy_src, copy_dst
        cus = torch.cuda.get_device_properties(dev).multi_processor_count
        extras["ceilings"] = ceilings_extra(args, dev, cus, 2 * S * inner * 2,
                                             2 * S_pad * inner * 2, relayout=(S, S_pad, 2 * H))
        extras["cfg5_prologue_qk"]["frac_of_best_relayout_stream"] = round(
            extras["cfg5_prologue_qk"]["gbps"] / extras["ceilings"]["relayout_stream"]["best_gbps"], 4)
        extras["cfg5_prologue_qk"]["frac_of_best_copy_stream"] = round(
            extras["cfg5_prologue_qk"]["gbps"] / extras["ceilings"]["copy_stream"]["best_gbps"], 4)
        extras["cfg4_dense_anchor_torch_sdpa"] = sdpa_anchor_extra(args, dev)
        extras["cfg3_qkv_proj"] = qkv_projection_extra(args, env=locals())
        extras["cfg3_attention_layer"] = attention_layer_extra(args, env=locals())
        for name in ("cfg3_1344x768x5s_frame0", "cfg2_864x480x7s", "cfg4_dense_864x480x7s",
                     "axial_h3_864x480x124"):
            sh = C.ALL[name]
            p = h3hip.TilePlan(sh.mask_rule(), heads=sh.heads)
            qq = torch.randn((sh.heads, p.seq_pad, D), generator=g, device=dev).to(torch.bfloat16)
            kk = torch.randn_like(qq)
            vv = torch.randn_like(qq)
            oo = torch.empty_like(qq)
            ms = interleaved_medians({"attn": lambda: ops.bsattn_fwd(p, qq, kk, vv, scale, out=oo)},
                                     reps=max(12, args.steps))["attn"]
            fl = p.nnz * sh.heads * FLOP_PER_TILE_HEAD
            extras[name] = {"timing": "median of 12+ calls", "attn_ms": round(ms, 4),
                            "active_tiles_per_head": p.nnz,
                            "density": round(p.density, 5),
                            "tflops_active": round(fl / (ms * 1e-3) / 1e12, 3),
                            "mfma_peak_frac": round(fl / (ms * 1e-3) / 1e12 / PEAK_BF16_TFLOPS, 4)}
            if sh.rule == "axial":
                kw = sh.oracle_rule_kwargs()
                extras[name]["heads"] = sh.heads
                extras[name]["token_density"] = round(h3hip.axial_token_density(
                    sh.prefix_len, sh.frames, sh.height, sh.width, kw["landmarks"]), 5)
            del qq, kk, vv, oo
            p.close()
        result["extras"] = extras
        # Against what the chip sustains for the kernel's MFMA shape on random
        # operands, measured in this run (the ceilings extra).
        c32 = extras["ceilings"]["mfma32_random_tflops"]
        result["attn_frac_of_same_run_mfma_stream"] = round(attn_tflops / c32, 4)

    if not args.no_cpu_baseline:
        result["cpu_baseline"] = cpu_baseline(shape, plan.tiles())
    print(json.dumps(result), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
