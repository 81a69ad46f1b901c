// The int8 projections' GEMM on four waves: tiles of W x^T, from one row up.
//
// The loop is the bf16 GEMM's (proj_gemm.hip has its layout and why it is four waves)
// with v_mfma_i32_16x16x64_i8 in place of the bf16 product: twice the operations for the
// same LDS bytes, loads and matrix-core cycles (gen_gemm_i8_loop.py). The 256 accumulators
// are int32 and exact. Rows of x past seq_len and of W past its last read as zeros, so
// a tile at either edge needs no case of its own before its stores.
//
// What bounds it: large products the chip's power limit (31,885 x 5,120 x 15,360 on random
// operands 1.86 ms, 2,690 TOP/s, on zeros 1.39; the library's int8 product of these sizes takes
// 2.07-2.13); few rows W's bytes (one token x 5,120 x 15,360 with norm 16.3-17.5 us, 4.5-4.8 TB/s
// with the launch) and, of a small W, the launch and 40 steps' latencies (one token x 5,120 x
// 5,120 7.1 us, 125 tokens 11.8).
//
// Epilogue: each sum to fp32, times its channel's and its token's scale, to bf16, into
// LDS as token rows, and from there what the bf16 projections do (proj_rows.h); in
// H3HIP_ROUND_ONCE Q and K go through LDS in fp32 (finish_tile_once). Beyond its
// reduction a 256 x 256 tile takes 9 us, with norm and rotation 14.
#pragma once

#include "gemm_i8_loop.inc"
#include "proj_i8.h"
#include "proj_i8_tile.h"
#include "proj_rows.h"
#include "tile_order.h"

namespace h3hip {

namespace {

constexpr int kWaves = H3_GEMM_I8_WAVES;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 128;               // reduction per step (bytes)

typedef f32x4 f32x4_any __attribute__((aligned(4)));   // scales of any first channel
typedef int i32x32 __attribute__((ext_vector_type(32)));
// A wave's accumulators, 8 blocks of 16 x 16 to a vector (the last may be part used).
template <int kNA, int kMB>
constexpr int kAccs = (kNA * kMB + 7) / 8;

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

#define H3_SCALARS                                                                          \
  [x_lo] "s"(x_lo), [x_hi] "s"(x_hi), [x_rec] "s"(x_rec), [w_lo] "s"(w_lo), [w_hi] "s"(w_hi), \
      [w_rec] "s"(w_rec), [steps] "s"(steps), [m0x] "s"(m0x), [m0w] "s"(m0w)

// One tile shape: its LDS and its reduction loop, from lane offsets and scalars
// to accumulators.
template <int kNA, int kMB, bool kPair>
struct Shape;
#define H3_SHAPE(NA, MB, PAIR, NAME)                                                         \
  template <>                                                                                \
  struct Shape<NA, MB, PAIR> {                                                                  \
    static constexpr int kLds = H3_GEMM_I8_LDS_##NAME, kBases = H3_GEMM_I8_BASES_##NAME;       \
    static __device__ __forceinline__ void reduce(i32x32 (&c)[kAccs<NA, MB>], const int* ra,   \
                                                  const int* rb, const int* xv, const int* wv, \
                                                  uint32_t x_lo, uint32_t x_hi, uint32_t x_rec, \
                                                  uint32_t w_lo, uint32_t w_hi, uint32_t w_rec, \
                                                  uint32_t steps, uint32_t m0x, uint32_t m0w) { \
      asm volatile(H3_GEMM_I8_LOOP_##NAME                                                    \
                   : H3_GEMM_I8_OUT_##NAME(c)                                                \
                   : H3_GEMM_I8_IN_##NAME(ra, rb, xv, wv), H3_SCALARS                        \
                   : H3_GEMM_I8_CLOBBERS_##NAME);                                            \
    }                                                                                        \
  };
H3_SHAPE(8, 8, false, 256x256)
H3_SHAPE(8, 7, false, 256x224)
H3_SHAPE(8, 6, false, 256x192)
H3_SHAPE(8, 5, false, 256x160)
H3_SHAPE(8, 4, false, 256x128)
H3_SHAPE(4, 6, false, 128x192)
H3_SHAPE(4, 5, false, 128x160)
H3_SHAPE(4, 4, false, 128x128)
H3_SHAPE(4, 4, true, 128x128p)
H3_SHAPE(4, 2, true, 128x64p)
H3_SHAPE(4, 1, true, 128x32p)
H3_SHAPE(2, 2, true, 64x64p)
H3_SHAPE(1, 2, true, 32x64p)
H3_SHAPE(1, 1, true, 32x32p)

// A lane's scales: of token 16 (kMB wt + mb) + lr, and of channels 16 (kNA wc + na) + 4g .. +3.
template <int kNA, int kMB>
struct Scales {
  float x[kMB];
  f32x4 w[kNA];
  // Past the last token or channel: the last one's, unused.
  __device__ __forceinline__ void load_x(const ProjI8Args& a, int wave, int lane, int m0) {
    const int wt = wave & 1, lr = lane & 15;
#pragma unroll
    for (int mb = 0; mb < kMB; mb++)
      x[mb] = a.x_scale[min(m0 + 16 * (kMB * wt + mb) + lr, a.out.seq_len - 1)];
  }
  __device__ __forceinline__ void load_w(const ProjI8Args& a, int wave, int lane, int n0) {
    const int wc = wave >> 1, g = lane >> 4;
    if (n0 + 32 * kNA <= a.n_total) {
#pragma unroll
      for (int na = 0; na < kNA; na++)
        w[na] = *reinterpret_cast<const f32x4_any*>(a.w_scale + n0 + 16 * (kNA * wc + na) + 4 * g);
      return;
    }
#pragma unroll
    for (int na = 0; na < kNA; na++) {
      const int n = n0 + 16 * (kNA * wc + na) + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; i++) w[na][i] = a.w_scale[min(n + i, a.n_total - 1)];
    }
  }
};

// Accumulators of channels 16 (kNA wc + na) + 4g .. +3 and token 16 (kMB wt + mb) + lr, with
// their scales. The channel's scale first: a weight's is moderate, a token's may be
// near either end of fp32, and so nothing overflows between that the result does not.
template <int kNA, int kMB>
__device__ __forceinline__ f32x4 scaled_sums(const i32x32 (&c)[kAccs<kNA, kMB>], int na, int mb,
                                             float xs, const f32x4& ws) {
  const int e = 4 * (kMB * na + mb);
  const i32x32& v = c[e / 32];
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] = (float)v[e % 32 + i] * ws[i] * xs;
  return y;
}
// The same rounded to bf16.
template <int kNA, int kMB>
__device__ __forceinline__ u32x2 scaled_block(const i32x32 (&c)[kAccs<kNA, kMB>], int na, int mb,
                                              float xs, const f32x4& ws) {
  const f32x4 y = scaled_sums<kNA, kMB>(c, na, mb, xs, ws);
  return u32x2{cvt_pk(y[0], y[1]), cvt_pk(y[2], y[3])};
}

// The epilogue of H3HIP_ROUND_ONCE for a tile that holds heads of Q or K: the scaled sums go
// to LDS as fp32 token rows, the head norm and the rotation read them there, and the one
// rounding to bf16 is the store's. An fp32 tile is twice a bf16 one's bytes, which the largest
// shapes' rings do not hold beside the rotation entries: such a tile goes in phases of
// kBlocks x 32 tokens, the accumulators of the later ones waiting in their registers. Against
// the bf16 rows of H3HIP_ROUND_FP32 a QKV call of 31,885 x 40 heads x 5,120 takes 0.8% more (2,077
// us), of 1,151 x 56 heads 0.7%, of one token nothing.
//
// 16-byte chunk c of a head's row l sits at c ^ (l & 15): the 16 rows that a block's write
// covers, and the two rows x 8 lanes of a read, are on 16 different chunks of a 256-byte bank
// window each.
template <int kNA, int kMB, bool kPair, int kHl>
__device__ __forceinline__ void finish_tile_once(const ProjI8Args& a, float* lds,
                                                 const i32x32 (&c)[kAccs<kNA, kMB>],
                                                 const Scales<kNA, kMB>& s, int wave, int lane,
                                                 int m0, int n0) {
  constexpr int kChannels = 32 * kNA, kHead = 128, kHeads = kChannels / kHead;
  constexpr int kBlockLds = 32 * kChannels * (int)sizeof(float);
  constexpr int kFit = (Shape<kNA, kMB, kPair>::kLds - kWaves * kRowTableLds) / kBlockLds;
  static_assert(kFit >= 1, "32 rows and the tables fit in the rings");
  constexpr int kPhases = (kMB + kFit - 1) / kFit, kBlocks = (kMB + kPhases - 1) / kPhases;
  const ProjArgs& o = a.out;
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
            scaled_sums<kNA, kMB>(c, na, mb0 + b, s.x[mb0 + b], s.w[na]);
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
template <int kNA, int kMB, bool kPair, int kMode, int kHl, bool kPlain, bool kOut>
__device__ __forceinline__ void finish_tile(const ProjI8Args& a, uint16_t* lds,
                                            const i32x32 (&c)[kAccs<kNA, kMB>],
                                            const Scales<kNA, kMB>& s, int wave, int lane, int m0,
                                            int n0) {
  constexpr int kTokens = 32 * kMB, kChannels = 32 * kNA;
  const int wc = wave >> 1, wt = wave & 1, lr = lane & 15, g = lane >> 4;
  if constexpr (kChannels < 128) {
    static_assert(kOut, "heads are written through LDS");
#pragma unroll
    for (int na = 0; na < kNA; na++) {
      const int64_t n = n0 + 16 * (kNA * wc + na) + 4 * g;
      if (n >= a.n_total) continue;
#pragma unroll
      for (int mb = 0; mb < kMB; mb++) {
        const int m = m0 + 16 * (kMB * wt + mb) + lr;
        if (m >= a.out.seq_len) continue;
        uint16_t* dst = a.out.q_out + (int64_t)m * a.out.ldo + n;
        const u32x2 y = scaled_block<kNA, kMB>(c, na, mb, s.x[mb], s.w[na]);
        if (n + 4 <= a.n_total) {
          *reinterpret_cast<u32x2_any*>(dst) = y;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (n + i < a.n_total) dst[i] = (uint16_t)(y[i / 2] >> (16 * (i & 1)));
        }
      }
    }
  } else {
    // The last token tile's workgroup also owns the rows behind its tile.
    auto zero_behind = [&]() __attribute__((always_inline)) {
      if (!kOut && m0 + kTokens >= a.out.seq_len)
        zero_rows<kChannels, kThreads>(a.out, 64 * wave + lane, m0 + kTokens, n0);
    };
    constexpr bool kOnce = kMode == H3HIP_ROUND_ONCE;
    if constexpr (kOnce) {
      if (n0 / 128 < 2 * a.out.heads) {   // a head of Q or K; V alone is stored as in any mode
        finish_tile_once<kNA, kMB, kPair, kHl>(a, reinterpret_cast<float*>(lds), c, s, wave, lane,
                                               m0, n0);
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
                                  4 * (g & 1)) = scaled_block<kNA, kMB>(c, na, mb, s.x[mb], s.w[na]);
    }
    __syncthreads();
    finish_tile_rows<kTokens, kChannels, kWaves, kMode, kHl, kPlain || kOnce, kOut, true>(
        a.out, lds, reinterpret_cast<RopeEntry*>(lds + kTokens * kChannels), wave, lane, m0, n0);
    zero_behind();
  }
}

template <int kNA, int kMB, bool kPair, int kMode, int kHl, bool kPlain, bool kOut>
__global__ __launch_bounds__(kThreads, kPair ? 2 : 1) void proj_i8_gemm_kernel(ProjI8Args a) {
  using S = Shape<kNA, kMB, kPair>;
  constexpr int kTokens = 32 * kMB, kChannels = 32 * kNA;
  static_assert(kChannels < 128 || S::kLds >= 2 * kTokens * kChannels + kWaves * kRowTableLds,
                "the epilogue's rows and tables fit in the rings");
  static_assert(!kPair || 2 * S::kLds <= 163840, "two workgroups' rings fit a CU");
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds / 2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wc = wave >> 1, wt = wave & 1;   // channel and token half of the tile
  const TileOrder order{a.out.tiles_m, (a.n_total + kChannels - 1) / kChannels, a.out.chunk};
  const int xcd = blockIdx.x % kOrderXcds, slot = blockIdx.x / kOrderXcds;
  if (slot >= order.length(xcd)) return;
  const uint32_t tile = order.tile(xcd, slot);
  const int m0 = (int)(tile >> 16) * kTokens, n0 = (int)(tile & 0xffff) * kChannels;

  const int lr = lane & 15, g = lane >> 4;
  const uint32_t lds_base = uniform((uint32_t)(size_t)(__attribute__((address_space(3))) uint16_t*)lds);
  int ra[2 * S::kBases], rb[2 * S::kBases], xv[kMB], wv[kNA];
#pragma unroll
  for (int b = 0; b < S::kBases; b++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int at = (int)lds_base + 65536 * b + (((4 * u + g) ^ p_swz(lr)) * 16);
      ra[2 * b + u] = at + (16 * kNA * wc + lr) * 128;
      rb[2 * b + u] = at + (16 * kMB * wt + lr) * 128;
    }
  const int ldx = (int)a.ldx, ldw = (int)a.ldw;
  auto load_offset = [&](int rows, int i, int ld) __attribute__((always_inline)) {
    const int r = rows * wave + 8 * i + (lane >> 3);
    return r * ld + (((lane & 7) ^ p_swz(r)) * 16) - 1024 * (i & 3);
  };
#pragma unroll
  for (int i = 0; i < kMB; i++) xv[i] = load_offset(8 * kMB, i, ldx);
#pragma unroll
  for (int i = 0; i < kNA; i++) wv[i] = load_offset(8 * kNA, i, ldw);
  const uint64_t xp = (uint64_t)(uintptr_t)(a.x + (int64_t)m0 * a.ldx);
  const uint64_t wp = (uint64_t)(uintptr_t)(a.w + (int64_t)n0 * a.ldw);
  const uint32_t x_lo = uniform((uint32_t)xp), x_hi = uniform((uint32_t)(xp >> 32));
  const uint32_t w_lo = uniform((uint32_t)wp), w_hi = uniform((uint32_t)(wp >> 32));
  // Bytes of the tile's rows that exist: what lies past them reads as zero.
  const int x_rows = min(a.out.seq_len - m0, kTokens), w_rows = min(a.n_total - n0, kChannels);
  const uint32_t x_rec = uniform((uint32_t)((x_rows - 1) * ldx + a.in));
  const uint32_t w_rec = uniform((uint32_t)((w_rows - 1) * ldw + a.in));
  const uint32_t steps = uniform((uint32_t)(a.in / kStep));
  const uint32_t m0w = uniform(lds_base + 1024u * kNA * wave);
  const uint32_t m0x = uniform(lds_base + 1024u * kMB * wave);
  // The scales arrive during the loop; the tokens' of the largest tile would be spilled
  // across it, and the channels' too where its epilogue goes in phases.
  constexpr bool kEarlyX = kNA * kMB < 64, kEarlyW = kEarlyX || kMode != H3HIP_ROUND_ONCE;
  Scales<kNA, kMB> scales;
  if (kEarlyX) scales.load_x(a, wave, lane, m0);
  if (kEarlyW) scales.load_w(a, wave, lane, n0);
  i32x32 c[kAccs<kNA, kMB>];
  S::reduce(c, ra, rb, xv, wv, x_lo, x_hi, x_rec, w_lo, w_hi, w_rec, steps, m0x, m0w);

  // The lane again, from the lane counter: kept from before the loop it would
  // be spilled across it.
  int lane2;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane2));
  if (!kEarlyX) scales.load_x(a, wave, lane2, m0);
  if (!kEarlyW) scales.load_w(a, wave, lane2, n0);
  finish_tile<kNA, kMB, kPair, kMode, kHl, kPlain, kOut>(a, lds, c, scales, wave, lane2, m0, n0);
}

// The launch order of a shape's tiles, into a, and the grid that runs it.
template <int kNA, int kMB>
dim3 order_grid(ProjI8Args& a) {
  const ProjGrid g = proj_i8_grid(a.out.seq_len, a.n_total, 32 * kMB, 32 * kNA);
  a.out.tiles_m = g.order.tiles_m;
  a.out.chunk = g.order.chunk;
  return dim3(kOrderXcds * g.longest);
}

inline int too_large(const ProjI8Args& a) {
  set_error("too many rows or channels for one launch (%d x %d)", a.out.seq_len, a.n_total);
  return H3HIP_EINVAL;
}

}  // namespace

}  // namespace h3hip
