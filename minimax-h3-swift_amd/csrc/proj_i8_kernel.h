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
#include "proj_finish.h"
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
  auto sums = [&](int na, int mb) __attribute__((always_inline)) {
    return scaled_sums<kNA, kMB>(c, na, mb, scales.x[mb], scales.w[na]);
  };
  finish_tile<kNA, kMB, S::kLds, kWaves, kMode, kHl, kPlain, kOut>(a.out, a.n_total, lds, sums, wave,
                                                                   lane2, m0, n0);
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
