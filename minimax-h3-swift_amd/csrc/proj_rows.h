// The second half of a projection's epilogue: the bf16 product, staged in LDS as
// token rows, to the outputs, with the head norm and the rotation on the way. Shared by
// the bf16 and the int8 projections (proj_gemm.hip, proj_i8_kernel.h), whose accumulators
// differ and whose rows do not.
#pragma once

#include <type_traits>

#include "norm_rope.h"
#include "proj.h"

namespace h3hip {

// Up to 8 channels of a token-major row, which may begin anywhere.
__device__ __forceinline__ void store_row_chunk(uint16_t* dst, u32x4 v, int left) {
  if (left >= 8) {
    *reinterpret_cast<u32x4_any*>(dst) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (e < left) dst[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
}

// Head hg of Q | K | V: its part's output, at the head.
template <class Args>
__device__ __forceinline__ uint16_t* head_rows(const Args& a, int hg) {
  const int part = hg / a.heads;
  uint16_t* out = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
  return out + (int64_t)(hg - part * a.heads) * a.seq_pad * 128;
}

// Zeros into rows m0 .. seq_pad - 1 of the heads of channels n0 .., by kThreads threads.
template <int kChannels, int kThreads, class Args>
__device__ __forceinline__ void zero_rows(const Args& a, int tid, int m0, int n0) {
  constexpr int kHead = 128, kChunks = kHead / 8;
#pragma unroll 1
  for (int hg = n0 / kHead; hg < min((n0 + kChannels) / kHead, 3 * a.heads); hg++) {
    uint16_t* head = head_rows(a, hg);
    for (int r = m0 + tid / kChunks; r < a.seq_pad; r += kThreads / kChunks)
      *reinterpret_cast<u32x4*>(head + (int64_t)r * kHead + 8 * (tid % kChunks)) =
          u32x4{0u, 0u, 0u, 0u};
  }
}

// Between a wave's LDS accesses that meet in other lanes: the hardware runs them in order, and
// this keeps the compiler from changing it. No instruction.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// The rotation entries of 8 token rows, from the table to the lanes of the prologue's
// row layout: lane j of row group rg needs entries 8j .. 8j + 7 of its row, 128 bytes
// (fp32; 64 in bf16) from its neighbour's. Loaded like that every load of a wave touches
// 64 lines, and the loads, not the arithmetic, took the epilogue's time: at 31,885 tokens x 40
// heads the fp32 norm and rotation added 16.6 us to a 256 x 256 tile. So the 8 lanes load 8
// (fp32) or 16 (bf16) consecutive entries at a time, whole lines, and trade them through 4 KiB
// of LDS of the wave's own: 6.2 us in fp32, of which 4.8 are its instructions; 10.8 in
// reference rounding (13.4 before), whose roundings are 1.5 times the instructions.
//
// Entry 8b + i of a row is at unit (i >> 1) ^ u(b) of its 64-byte block b ^ rg, with u(b) =
// (b >> 2 & 1) | (rg & 1) << 1: 32 lanes writing one entry each, or 16 reading two, then meet
// in every bank once.
template <int kMode, int kHl>
struct RowTable {
  static constexpr bool kRef = kMode == H3HIP_ROUND_REFERENCE;
  static constexpr int kLoads = kRef ? kHl / 2 : kHl;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  u32x4 ref[kRef ? kLoads : 1];
  f32x4 f32[kRef ? 1 : kLoads];

  __device__ __forceinline__ void load(const void* table, int64_t row, int j) {
    constexpr int kHalf = 8 * kHl;
    if constexpr (kRef) {
      const uint16_t* p = static_cast<const uint16_t*>(table) + (row * kHalf + 2 * j) * 4;
#pragma unroll
      for (int t = 0; t < kLoads; t++) ref[t] = *reinterpret_cast<const u32x4*>(p + 64 * t);
    } else {
      const f32x4* p = static_cast<const f32x4*>(table) + row * kHalf + j;
#pragma unroll
      for (int t = 0; t < kLoads; t++) f32[t] = p[8 * t];
    }
  }
  static __device__ __forceinline__ int unit(int b, int rg) { return ((b >> 2) & 1) | (rg & 1) << 1; }
  // From the loaded registers to tab, through the wave's lds; the pairs of pair lanes.
  __device__ __forceinline__ void trade(RopeEntry* lds, int j, int rg, RopeEntry (&tab)[8]) {
    RopeEntry* mine = lds + 64 * rg;
    wave_lds_order();   // the last pass's reads
#pragma unroll
    for (int t = 0; t < kLoads; t++) {
      if constexpr (kRef) {   // entries 16t + 2j, + 1: (c, -s, s, c) bf16 each
        const int b = 2 * t + (j >> 2);
        const f32x4 v = {bf16_lo(ref[t][0]), bf16_lo(ref[t][1]), bf16_lo(ref[t][2]),
                         bf16_lo(ref[t][3])};
        *reinterpret_cast<f32x4*>(mine + 8 * (b ^ rg) + 2 * ((j & 3) ^ unit(b, rg))) = v;
      } else {                // entry 8t + j
        const f32x2 v = {f32[t][0], f32[t][2]};
        *reinterpret_cast<f32x2*>(mine + 8 * (t ^ rg) + 2 * ((j >> 1) ^ unit(t, rg)) + (j & 1)) = v;
      }
    }
    wave_lds_order();
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(mine + 8 * (j ^ rg) + 2 * (q ^ unit(j, rg)));
      tab[2 * q] = RopeEntry{v[0], v[1]};
      tab[2 * q + 1] = RopeEntry{v[2], v[3]};
    }
  }
};
constexpr int kRowTableLds = 8 * 64 * sizeof(RopeEntry);   // bytes of a wave

// Rows of kChannels in LDS, chunk c (16 bytes) of row r at c ^ e_swz(r) within its
// head, to the outputs. Each of kRowWaves waves takes whole rows, 8 at a time in the
// prologue's 8-lane layout, head after head, so that a row's rotation entries are
// fetched once. kHl = rot / 16 (8-channel chunks per rotation half);
// kPlain: every part unchanged; kOut: token-major with row stride ldo. kAnyWidth, with
// kOut: any output width, row stride and address; by heads: a tile of two heads may hold
// the last of one part and the first of the next, or only one. tables: kRowTableLds bytes
// for each wave.
template <int kTokens, int kChannels, int kRowWaves, int kMode, int kHl, bool kPlain, bool kOut,
          bool kAnyWidth = false, class Args>
__device__ __forceinline__ void finish_tile_rows(const Args& a, const uint16_t* lds,
                                                 RopeEntry* tables, int wave, int lane, int m0,
                                                 int n0) {
  constexpr int kHead = 128;
  constexpr int kHeads = kChannels / kHead, kRows = kTokens / kRowWaves;
  constexpr bool kRagged = kOut && kAnyWidth;
  static_assert(kRows % 8 == 0, "whole passes");
  const int row0 = kRows * wave;
  constexpr bool kFull = kHl == 8;
  const int j = lane & 7, rg = lane >> 3;
  const bool pair_lane = kFull || j < kHl;
  const int chunk_a = pair_lane ? j : 2 * kHl + 2 * (j - kHl);
  const int chunk_b = pair_lane ? j + kHl : chunk_a + 1;
  // Whether every channel of the tile is a channel of the output.
  const bool full = !kRagged || n0 + kChannels <= a.n_out;
  // Passes of 8 rows; head-major rows end at seq_pad, a multiple of 8.
  const int passes = kOut ? kRows / 8 : min(kRows, max(a.seq_pad - m0 - row0, 0)) / 8;
  const bool whole = m0 + row0 + kRows <= a.seq_len;
  // `count` heads of one part, from the tile's head nh0 on.
  auto finish_heads = [&](int nh0, auto count) __attribute__((always_inline)) {
    constexpr int kCount = decltype(count)::value;
    const int hg = n0 / kHead + nh0;
    const int part = kOut ? 0 : hg / a.heads;
    uint16_t* out = kOut ? a.q_out + n0 + nh0 * kHead : head_rows(a, hg);
    // This lane's two chunks of row r of the tile and head nh0 + nh.
    auto load_row = [&](int r, int nh, u32x4& oa, u32x4& ob) __attribute__((always_inline)) {
      const uint16_t* row = lds + r * kChannels + (nh0 + nh) * kHead;
      oa = *reinterpret_cast<const u32x4*>(row + ((chunk_a ^ e_swz(r & 15)) * 8));
      ob = *reinterpret_cast<const u32x4*>(row + ((chunk_b ^ e_swz(r & 15)) * 8));
    };
    auto store_row = [&](int r, int nh, bool valid, u32x4 oa,
                         u32x4 ob) __attribute__((always_inline)) {
      const int m = m0 + r;
      if (!valid) oa = ob = u32x4{0u, 0u, 0u, 0u};
      uint16_t* dst = kOut ? out + (int64_t)m * a.ldo + nh * kHead
                           : out + ((int64_t)nh * a.seq_pad + m) * kHead;
      if (kRagged && !full) {
        if (valid) {
          const int left = a.n_out - n0 - (nh0 + nh) * kHead;
          store_row_chunk(dst + 8 * chunk_a, oa, left - 8 * chunk_a);
          store_row_chunk(dst + 8 * chunk_b, ob, left - 8 * chunk_b);
        }
      } else if (!kOut || valid) {
        using Chunk = std::conditional_t<kRagged, u32x4_any, u32x4>;
        *reinterpret_cast<Chunk*>(dst + 8 * chunk_a) = oa;
        *reinterpret_cast<Chunk*>(dst + 8 * chunk_b) = ob;
      }
    };
    auto copy_rows = [&](int n, auto all_valid) __attribute__((always_inline)) {
#pragma unroll 2
      for (int pass = 0; pass < n; pass++) {
        const int r = row0 + 8 * pass + rg;
        const bool valid = decltype(all_valid)::value || m0 + r < a.seq_len;
#pragma unroll
        for (int nh = 0; nh < kCount; nh++) {
          u32x4 oa, ob;
          load_row(r, nh, oa, ob);
          store_row(r, nh, valid, oa, ob);
        }
      }
    };
    if constexpr (!kPlain && !kOut) {
      if (part < 2) {
        float gam[16];
        const uint16_t* gsrc = part == 0 ? a.q_gamma : a.k_gamma;
        unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_a), gam);
        unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_b), gam + 8);
        RopeEntry* mine = tables + 512 * wave;
        RowTable<kMode, kHl> table;
        auto fetch = [&](int pass) __attribute__((always_inline)) {
          table.load(a.table, min(m0 + row0 + 8 * pass + rg, a.seq_len - 1), j);
        };
        if (passes > 0) fetch(0);
        for (int pass = 0; pass < passes; pass++) {
          const int r = row0 + 8 * pass + rg;
          const bool valid = m0 + r < a.seq_len;
          RopeEntry tab[8];
          table.trade(mine, j, rg, tab);
          fetch(pass + 1);   // past the last pass: a row of the table, unused
#pragma unroll
          for (int nh = 0; nh < kCount; nh++) {
            u32x4 oa, ob;
            load_row(r, nh, oa, ob);
            float xr[16];
            unpack8(oa, xr);
            unpack8(ob, xr + 8);
            norm_rope<kMode, kFull>(xr, gam, pair_lane, tab, a.eps, oa, ob);
            store_row(r, nh, valid, oa, ob);
          }
        }
        return;
      }
    }
    if (whole)
      copy_rows(kRows / 8, std::true_type{});
    else
      copy_rows(passes, std::false_type{});
  };
  using One = std::integral_constant<int, 1>;
  if constexpr (kAnyWidth && !kOut && kHeads == 2) {
    const int hg = n0 / kHead;
    if (hg / a.heads != (hg + 1) / a.heads) {
#pragma unroll 1
      for (int nh = 0; nh < 2 && hg + nh < 3 * a.heads; nh++) finish_heads(nh, One{});
      return;
    }
  }
  finish_heads(0, std::integral_constant<int, kHeads>{});
}

}  // namespace h3hip
