// The second half of a projection's epilogue: the bf16 product, staged in LDS as
// token rows, to the outputs, with the head norm and the rotation on the way.
// Shared by the bf16 and the int8 projections (proj_gemm.hip, proj_i8.hip,
// proj_i8_gemm.hip), whose accumulators differ and whose rows do not.
#pragma once

#include <type_traits>

#include "norm_rope.h"
#include "proj.h"

namespace h3hip {

// Up to 8 channels of a token-major row; wide: the address is 16-byte aligned.
__device__ __forceinline__ void store_row_chunk(uint16_t* dst, u32x4 v, int left, bool wide) {
  if (wide && left >= 8) {
    *reinterpret_cast<u32x4*>(dst) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (e < left) dst[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
}

// Zeros into rows m0 .. of the heads of channels n0 ..: a tile of padding rows only.
template <int kTokens, int kChannels, int kThreads>
__device__ __forceinline__ void zero_tile_rows(const ProjArgs& a, int tid, int m0, int n0) {
  constexpr int kHead = 128, kChunks = kHead / 8;
  const int inner = a.heads * kHead, part = n0 / inner;
  const int head0 = (n0 - part * inner) / kHead;
  uint16_t* out = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
  for (int i = tid; i < kTokens * (kChannels / 8); i += kThreads) {
    const int head = head0 + i / (kTokens * kChunks), r = i / kChunks % kTokens;
    if (m0 + r < a.seq_pad)
      *reinterpret_cast<u32x4*>(out + ((int64_t)head * a.seq_pad + m0 + r) * kHead +
                                8 * (i % kChunks)) = u32x4{0u, 0u, 0u, 0u};
  }
}

// Rows of kChannels in LDS, chunk c (16 bytes) of row r at c ^ e_swz(r) within its
// head. Each of kRowWaves waves takes whole rows of one head, 8 at a time in the
// prologue's 8-lane layout. kHl = rot / 16 (8-channel chunks per rotation half);
// kPlain: every part unchanged; kOut: token-major with row stride ldo; kRagged (with
// kOut): any output width and row stride, wide saying that the row stride and the
// output's address allow 16-byte stores.
template <int kTokens, int kChannels, int kRowWaves, int kMode, int kHl, bool kPlain, bool kOut,
          bool kRagged = false>
__device__ __forceinline__ void finish_tile_rows(const ProjArgs& a, const uint16_t* lds, int wave,
                                                 int lane, int m0, int n0, bool wide = true) {
  constexpr int kHead = 128;
  constexpr int kHeads = kChannels / kHead, kRows = kTokens * kHeads / kRowWaves;
  static_assert(kRows % 8 == 0 && (kHeads == 1 || (kHeads == 2 && kRowWaves == 4)),
                "whole passes of one head a wave");
  const int nh = kHeads == 2 ? wave >> 1 : 0;
  const int row0 = kRows * (kHeads == 2 ? wave & 1 : wave);
  const int inner = a.heads * kHead;
  const int part = kOut ? 0 : n0 / inner;
  const int head = kOut ? 0 : (n0 - part * inner) / kHead + nh;
  uint16_t* out = part == 0 ? a.q_out : part == 1 ? a.k_out : a.v_out;
  const bool norm = !kPlain && !kOut && part < 2;
  constexpr bool kFull = kHl == 8;
  constexpr int kHalf = 8 * kHl;
  const int j = lane & 7, rg = lane >> 3;
  const bool pair_lane = kFull || j < kHl;
  const int chunk_a = pair_lane ? j : 2 * kHl + 2 * (j - kHl);
  const int chunk_b = pair_lane ? j + kHl : chunk_a + 1;
  float gam[16];
  if (norm) {
    const uint16_t* gsrc = part == 0 ? a.q_gamma : a.k_gamma;
    unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_a), gam);
    unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_b), gam + 8);
  }
  // Row r of the tile: this lane's two chunks, normalised and rotated.
  auto finish_row = [&](int r, auto whole, auto rotated) __attribute__((always_inline)) {
    const int m = m0 + r;
    const bool valid = decltype(whole)::value || m < a.seq_len;
    const uint16_t* row = lds + r * kChannels + nh * kHead;
    u32x4 oa = *reinterpret_cast<const u32x4*>(row + ((chunk_a ^ e_swz(r & 15)) * 8));
    u32x4 ob = *reinterpret_cast<const u32x4*>(row + ((chunk_b ^ e_swz(r & 15)) * 8));
    if constexpr (decltype(rotated)::value) {
      RopeEntry tab[8];
      const int64_t entry = (int64_t)(decltype(whole)::value ? m : min(m, a.seq_len - 1)) * kHalf +
                            (pair_lane ? 8 * j : 0);
      if (kMode == H3HIP_ROUND_REFERENCE) {
        const u32x4* tp =
            reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.table) + entry * 4);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const u32x4 tv = tp[q];   // (c, -s, s, c) bf16 of pairs 2q, 2q + 1
          tab[2 * q] = RopeEntry{bf16_lo(tv[0]), bf16_lo(tv[1])};
          tab[2 * q + 1] = RopeEntry{bf16_lo(tv[2]), bf16_lo(tv[3])};
        }
      } else {
        const f32x4* tp = reinterpret_cast<const f32x4*>(a.table) + entry;
#pragma unroll
        for (int e = 0; e < 8; e++) tab[e] = RopeEntry{tp[e][0], tp[e][2]};
      }
      float xr[16];
      unpack8(oa, xr);
      unpack8(ob, xr + 8);
      norm_rope<kMode, kFull>(xr, gam, pair_lane, tab, a.eps, oa, ob);
    }
    if (!valid) oa = ob = u32x4{0u, 0u, 0u, 0u};
    uint16_t* dst = kOut ? a.q_out + (int64_t)m * a.ldo + n0 + nh * kHead
                         : out + ((int64_t)head * a.seq_pad + m) * kHead;
    if constexpr (kRagged) {
      if (valid) {
        const int left = a.n_out - n0 - nh * kHead;
        store_row_chunk(dst + 8 * chunk_a, oa, left - 8 * chunk_a, wide);
        store_row_chunk(dst + 8 * chunk_b, ob, left - 8 * chunk_b, wide);
      }
    } else if (!kOut || valid) {
      *reinterpret_cast<u32x4*>(dst + 8 * chunk_a) = oa;
      *reinterpret_cast<u32x4*>(dst + 8 * chunk_b) = ob;
    }
  };
  // Passes of 8 rows; head-major rows end at seq_pad, a multiple of 8.
  const int passes = kOut ? kRows / 8 : min(kRows, max(a.seq_pad - m0 - row0, 0)) / 8;
  auto finish_rows = [&](auto whole, auto rotated) __attribute__((always_inline)) {
    if constexpr (decltype(whole)::value) {
#pragma unroll 2
      for (int pass = 0; pass < kRows / 8; pass++) finish_row(row0 + 8 * pass + rg, whole, rotated);
    } else {
      for (int pass = 0; pass < passes; pass++) finish_row(row0 + 8 * pass + rg, whole, rotated);
    }
  };
  const bool whole = m0 + row0 + kRows <= a.seq_len;
  if constexpr (!kPlain && !kOut) {
    if (norm) {
      if (whole)
        finish_rows(std::true_type{}, std::true_type{});
      else
        finish_rows(std::false_type{}, std::true_type{});
      return;
    }
  }
  if (whole)
    finish_rows(std::true_type{}, std::false_type{});
  else
    finish_rows(std::false_type{}, std::false_type{});
}

}  // namespace h3hip
