// The epilogue of a projection's tile on four waves, from the sums in a wave's registers to
// the outputs: shared by the int8 and the 4-bit projections (proj_i8_kernel.h,
// proj_mx4_kernel.h), whose products differ and whose tiles do not.
//
// sums(na, mb): channels 16 (kNA wc + na) + 4g .. +3 of token 16 (kMB wt + mb) + lr, in fp32,
// with wc = wave >> 1, wt = wave & 1, lr = lane & 15, g = lane >> 4. kLds: bytes of LDS that the
// reduction no longer needs.
#pragma once

#include <type_traits>

#include "proj_rows.h"

namespace h3hip {

// The epilogue of H3HIP_ROUND_ONCE for a tile that holds heads of Q or K: the sums go
// to LDS as fp32 token rows, the head norm and the rotation read them there, and the one
// rounding to bf16 is the store's. An fp32 tile is twice a bf16 one's bytes, which the largest
// shapes' rings do not hold beside the rotation entries: such a tile goes in phases of
// kBlocks x 32 tokens, the accumulators of the later ones waiting in their registers. Against
// the bf16 rows of H3HIP_ROUND_FP32 a QKV call of 31,885 x 40 heads x 5,120 takes 0.8% more (2,077
// us), of 1,151 x 56 heads 0.7%, of one token nothing (int8; on 4-bit operands, whose loop is half as
// long, 4% on 256 x 256: 1,273 -> 1,323 us; on the 256 x 224 that is picked less than nothing, 1,269 ->
// 1,247 in turn, and 1,124 without norm and rotation).
//
// 16-byte chunk c of a head's row l sits at c ^ (l & 15): the 16 rows that a block's write
// covers, and the two rows x 8 lanes of a read, are on 16 different chunks of a 256-byte bank
// window each.
template <int kNA, int kMB, int kLds, int kWaves, int kHl, class Args, class Sums>
__device__ __forceinline__ void finish_tile_once(const Args& o, float* lds, const Sums& sums,
                                                 int wave, int lane, int m0, int n0) {
  constexpr int kChannels = 32 * kNA, kHead = 128, kHeads = kChannels / kHead;
  constexpr int kBlockLds = 32 * kChannels * (int)sizeof(float);
  constexpr int kFit = (kLds - kWaves * kRowTableLds) / kBlockLds;
  static_assert(kFit >= 1, "32 rows and the tables fit in the rings");
  constexpr int kPhases = (kMB + kFit - 1) / kFit, kBlocks = (kMB + kPhases - 1) / kPhases;
  const int wc = wave >> 1, wt = wave & 1, lr = lane & 15, g = lane >> 4;
  const int j = lane & 7, rg = lane >> 3;
  constexpr bool kFull = kHl == 8;
  const bool pair_lane = kFull || j < kHl;
  const int chunk_a = pair_lane ? j : 2 * kHl + 2 * (j - kHl);
  const int chunk_b = pair_lane ? j + kHl : chunk_a + 1;
  RopeEntry* mine = reinterpret_cast<RopeEntry*>(lds + kBlocks * kBlockLds / (int)sizeof(float)) +
                    512 * wave;
  const int hg0 = n0 / kHead;
  const bool one_part = kHeads == 1 || hg0 / o.heads == (hg0 + 1) / o.heads;

#pragma unroll
  for (int phase = 0; phase < kPhases; phase++) {
    const int mb0 = kBlocks * phase, blocks = min(kBlocks, kMB - mb0);
    if (phase > 0) __syncthreads();   // the last phase's rows are read
#pragma unroll
    for (int na = 0; na < kNA; na++) {
      const int at = 4 * (kNA * wc + na) + g;   // the tile's 16-byte chunk of these channels
      const int pos = (at & ~31) | ((at & 31) ^ lr);
#pragma unroll
      for (int b = 0; b < blocks; b++)
        *reinterpret_cast<f32x4*>(lds + (16 * (blocks * wt + b) + lr) * kChannels + 4 * pos) =
            sums(na, mb0 + b);
    }
    __syncthreads();
    // A wave takes 8 x blocks consecutive rows, 8 at a time: tokens from m1 on.
    const int l0 = 8 * blocks * wave;
    const int m1 = m0 + 16 * (kMB * (wave >> 1) + mb0) + 8 * blocks * (wave & 1);
    const int passes = min(8 * blocks, max(o.seq_pad - m1, 0)) / 8;
    auto finish_heads = [&](int nh0, auto count) __attribute__((always_inline)) {
      constexpr int kCount = decltype(count)::value;
      const int part = (hg0 + nh0) / o.heads;
      uint16_t* out = head_rows(o, hg0 + nh0);
      auto load_row = [&](int l, int nh, float (&x)[16]) __attribute__((always_inline)) {
        const float* row = lds + l * kChannels + (nh0 + nh) * kHead;
#pragma unroll
        for (int h = 0; h < 4; h++) {
          const int chunk = 2 * (h < 2 ? chunk_a : chunk_b) + (h & 1);
          const f32x4 v = *reinterpret_cast<const f32x4*>(row + 4 * (chunk ^ (l & 15)));
#pragma unroll
          for (int i = 0; i < 4; i++) x[4 * h + i] = v[i];
        }
      };
      auto store_row = [&](int m, int nh, u32x4 oa, u32x4 ob) __attribute__((always_inline)) {
        if (m >= o.seq_len) oa = ob = u32x4{0u, 0u, 0u, 0u};
        uint16_t* dst = out + ((int64_t)nh * o.seq_pad + m) * kHead;
        *reinterpret_cast<u32x4*>(dst + 8 * chunk_a) = oa;
        *reinterpret_cast<u32x4*>(dst + 8 * chunk_b) = ob;
      };
      if (part == 2) {   // beside K's last head: rounded and stored
        for (int pass = 0; pass < passes; pass++) {
          const int r = 8 * pass + rg;
#pragma unroll
          for (int nh = 0; nh < kCount; nh++) {
            float x[16];
            load_row(l0 + r, nh, x);
            store_row(m1 + r, nh, pack8(x), pack8(x + 8));
          }
        }
        return;
      }
      float gam[16];
      const uint16_t* gsrc = part == 0 ? o.q_gamma : o.k_gamma;
      unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_a), gam);
      unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_b), gam + 8);
      RowTable<H3HIP_ROUND_ONCE, kHl> table;
      auto fetch = [&](int pass) __attribute__((always_inline)) {
        table.load(o.table, min(m1 + 8 * pass + rg, o.seq_len - 1), j);
      };
      if (passes > 0) fetch(0);
      for (int pass = 0; pass < passes; pass++) {
        const int r = 8 * pass + rg;
        RopeEntry tab[8];
        table.trade(mine, j, rg, tab);
        fetch(pass + 1);   // past the last pass: a row of the table, unused
#pragma unroll
        for (int nh = 0; nh < kCount; nh++) {
          float x[16];
          load_row(l0 + r, nh, x);
          u32x4 oa, ob;
          norm_rope<H3HIP_ROUND_ONCE, kFull>(x, gam, pair_lane, tab, o.eps, oa, ob);
          store_row(m1 + r, nh, oa, ob);
        }
      }
    };
    if (one_part) {
      finish_heads(0, std::integral_constant<int, kHeads>{});
    } else {   // the last head of Q or K and the first of the part behind it
#pragma unroll 1
      for (int nh = 0; nh < 2; nh++)
        finish_heads(nh, std::integral_constant<int, 1>{});
    }
  }
}

// The tile's epilogue. Tiles of a head or two go through LDS as token rows; narrower ones,
// whose few rows gain nothing from that, are stored from the accumulators, 32 bytes of a
// row at a time.
template <int kNA, int kMB, int kLds, int kWaves, int kMode, int kHl, bool kPlain, bool kOut,
          class Args, class Sums>
__device__ __forceinline__ void finish_tile(const Args& o, int n_total, uint16_t* lds,
                                            const Sums& sums, int wave, int lane, int m0, int n0) {
  constexpr int kThreads = 64 * kWaves;
  auto block = [&](int na, int mb) __attribute__((always_inline)) {   // rounded to bf16
    const f32x4 y = sums(na, mb);
    return u32x2{cvt_pk(y[0], y[1]), cvt_pk(y[2], y[3])};
  };
  constexpr int kTokens = 32 * kMB, kChannels = 32 * kNA;
  const int wc = wave >> 1, wt = wave & 1, lr = lane & 15, g = lane >> 4;
  if constexpr (kChannels < 128) {
    static_assert(kOut, "heads are written through LDS");
#pragma unroll
    for (int na = 0; na < kNA; na++) {
      const int64_t n = n0 + 16 * (kNA * wc + na) + 4 * g;
      if (n >= n_total) continue;
#pragma unroll
      for (int mb = 0; mb < kMB; mb++) {
        const int m = m0 + 16 * (kMB * wt + mb) + lr;
        if (m >= o.seq_len) continue;
        uint16_t* dst = o.q_out + (int64_t)m * o.ldo + n;
        const u32x2 y = block(na, mb);
        if (n + 4 <= n_total) {
          *reinterpret_cast<u32x2_any*>(dst) = y;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (n + i < n_total) dst[i] = (uint16_t)(y[i / 2] >> (16 * (i & 1)));
        }
      }
    }
  } else {
    // The last token tile's workgroup also owns the rows behind its tile.
    auto zero_behind = [&]() __attribute__((always_inline)) {
      if (!kOut && m0 + kTokens >= o.seq_len)
        zero_rows<kChannels, kThreads>(o, 64 * wave + lane, m0 + kTokens, n0);
    };
    constexpr bool kOnce = kMode == H3HIP_ROUND_ONCE;
    if constexpr (kOnce) {
      if (n0 / 128 < 2 * o.heads) {   // a head of Q or K; V alone is stored as in any mode
        finish_tile_once<kNA, kMB, kLds, kWaves, kHl>(o, reinterpret_cast<float*>(lds), sums, wave,
                                                      lane, m0, n0);
        zero_behind();
        return;
      }
    }
    // bf16 token rows of the whole tile in LDS; chunk c (16 bytes) of row r sits
    // at c ^ e_swz(r), within its head.
#pragma unroll
    for (int na = 0; na < kNA; na++) {
      const int chunk = 2 * (kNA * wc + na) + (g >> 1);
      const int pos = (chunk & 16) | ((chunk & 15) ^ e_swz(lr));
#pragma unroll
      for (int mb = 0; mb < kMB; mb++)
        *reinterpret_cast<u32x2*>(lds + (16 * (kMB * wt + mb) + lr) * kChannels + pos * 8 +
                                  4 * (g & 1)) = block(na, mb);
    }
    __syncthreads();
    finish_tile_rows<kTokens, kChannels, kWaves, kMode, kHl, kPlain || kOnce, kOut, true>(
        o, lds, reinterpret_cast<RopeEntry*>(lds + kTokens * kChannels), wave, lane, m0, n0);
    zero_behind();
  }
}

}  // namespace h3hip
