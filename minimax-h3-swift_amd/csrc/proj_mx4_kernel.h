// The 4-bit projections' GEMM on four waves: tiles of W x^T, from one row up.
//
//   y[m, n] = sum over blocks b of 32 of 2^(ex[m, b] + ew[n, b]) sum_i x[m, i] w[n, i]
//
// The loop is the bf16 GEMM's (proj_gemm.hip has its layout and why it is four waves) with
// v_mfma_scale_f32_16x16x128_f8f6f4 on e2m1 operands in place of the bf16 product: four times the
// operations for the same LDS bytes, loads and matrix-core cycles (gen_gemm_mx4_loop.py). A
// lane's 16 bytes of a row are one block of 32, so the block's scale is a byte of a register of
// that lane, and the scales of 16 rows and two steps are one load of 256 bytes in lane order.
// Products of values are exact; the sums are fp32 in the matrix core, in the order of k, which
// does not depend on the tile: a row's bits are the same in every call. Rows of x past seq_len
// and of W past its last read as zeros, so a tile at either edge needs no case of its own before
// its stores.
//
// Epilogue: proj_finish.h, on the sums as they are.
//
// What bounds it: large products the chip's power limit (31,885 x 5,120 x 5,120 393-445 us by card
// and warmth, 3,760 to 4,250 TFLOP/s, matrix cores busy 53% of the cycles at 1.8 GHz; a stream of the instruction alone 7,090; a
// step of a 256 x 256 tile 1.59 us on Gaussians and 1.31 on zeros), 637 x 1,000 x 777 the latency of its four
// steps (4.8 us). Two workgroups of 128 x 192 a CU, whose loops cover each other's epilogues, are bound by
// their LDS reads: 449 us.
#pragma once

#include "gemm_mx4_loop.inc"
#include "proj_mx4.h"
#include "proj_mx4_tile.h"
#include "proj_finish.h"
#include "tile_order.h"

namespace h3hip {

namespace {

constexpr int kWaves = H3_GEMM_MX4_WAVES;
constexpr int kThreads = 64 * kWaves;
constexpr int kStep = 128;               // bytes of a row per step: 256 values

typedef float f32x32 __attribute__((ext_vector_type(32)));
// A wave's accumulators, 8 blocks of 16 x 16 to a vector (the last may be part used).
template <int kNA, int kMB>
constexpr int kAccs = (kNA * kMB + 7) / 8;

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// Uniform operands of a reduction: the operands' first rows, the bytes that exist from there,
// LDS addresses of this wave's loads; of the scales the first of this wave's 16-row blocks,
// the bytes behind it and the bytes to the next pair of steps.
struct Scalars {
  uint32_t x_lo, x_hi, x_rec, w_lo, w_hi, w_rec, steps, m0x, m0w;
  uint32_t xs_lo, xs_hi, xs_rec, xs_step, ws_lo, ws_hi, ws_rec, ws_step, pairs;
};
#define H3_SCALARS                                                                          \
  [x_lo] "s"(s.x_lo), [x_hi] "s"(s.x_hi), [x_rec] "s"(s.x_rec), [w_lo] "s"(s.w_lo),         \
      [w_hi] "s"(s.w_hi), [w_rec] "s"(s.w_rec), [steps] "s"(s.steps), [m0x] "s"(s.m0x),     \
      [m0w] "s"(s.m0w), [xs_lo] "s"(s.xs_lo), [xs_hi] "s"(s.xs_hi), [xs_rec] "s"(s.xs_rec), \
      [xs_step] "s"(s.xs_step), [ws_lo] "s"(s.ws_lo), [ws_hi] "s"(s.ws_hi),                 \
      [ws_rec] "s"(s.ws_rec), [ws_step] "s"(s.ws_step), [pairs] "s"(s.pairs)

// One tile shape: its LDS and its reduction loop, from lane offsets and scalars
// to accumulators.
template <int kNA, int kMB, bool kPair>
struct Shape;
#define H3_SHAPE(NA, MB, PAIR, NAME)                                                         \
  template <>                                                                                \
  struct Shape<NA, MB, PAIR> {                                                                  \
    static constexpr int kLds = H3_GEMM_MX4_LDS_##NAME, kBases = H3_GEMM_MX4_BASES_##NAME;       \
    static __device__ __forceinline__ void reduce(f32x32 (&c)[kAccs<NA, MB>], const int* ra,   \
                                                  const int* rb, const int* xv, const int* wv, \
                                                  const int* sv, const Scalars& s) {           \
      asm volatile(H3_GEMM_MX4_LOOP_##NAME                                                    \
                   : H3_GEMM_MX4_OUT_##NAME(c)                                                \
                   : H3_GEMM_MX4_IN_##NAME(ra, rb, xv, wv, sv), H3_SCALARS                   \
                   : H3_GEMM_MX4_CLOBBERS_##NAME);                                            \
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

// Accumulators of channels 16 (kNA wc + na) + 4g .. +3 and token 16 (kMB wt + mb) + lr. Read
// one by one: the compiler has no copy of a whole vector of them.
template <int kNA, int kMB>
__device__ __forceinline__ f32x4 block_sums(const f32x32 (&c)[kAccs<kNA, kMB>], int na, int mb) {
  const int e = 4 * (kMB * na + mb);
  const f32x32& v = c[e / 32];
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; i++)
    asm("v_accvgpr_read_b32 %0, %1" : "=v"(y[i]) : "a"(v[e % 32 + i]));
  return y;
}

// A ProjMx4Args as the kernel and its epilogue take it: a launch of 128 bytes of arguments and
// more takes the host 0.9 us longer.
struct ProjMx4Packed {
  const uint8_t* __restrict__ x;
  const uint8_t* __restrict__ w;
  const uint8_t* __restrict__ x_scale;
  const uint8_t* __restrict__ w_scale;
  uint16_t* __restrict__ q_out;
  uint16_t* __restrict__ k_out;
  union {
    uint16_t* v_out;
    int64_t ldo;                           // of token rows
  };
  const uint16_t* __restrict__ q_gamma;
  const uint16_t* __restrict__ k_gamma;
  const void* __restrict__ table;
  int32_t ldx, ldw, in, n_out, seq_len, seq_pad, heads, tiles_m, chunk;
  float eps;
};

template <int kNA, int kMB, bool kPair, int kMode, int kHl, bool kPlain, bool kOut>
__global__ __launch_bounds__(kThreads, kPair ? 2 : 1) void proj_mx4_gemm_kernel(ProjMx4Packed a) {
  using S = Shape<kNA, kMB, kPair>;
  constexpr int kTokens = 32 * kMB, kChannels = 32 * kNA;
  static_assert(kChannels < 128 || S::kLds >= 2 * kTokens * kChannels + kWaves * kRowTableLds,
                "the epilogue's rows and tables fit in the rings");
  static_assert(!kPair || 2 * S::kLds <= 163840, "two workgroups' rings fit a CU");
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds / 2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wc = wave >> 1, wt = wave & 1;   // channel and token half of the tile
  const TileOrder order{a.tiles_m, (a.n_out + kChannels - 1) / kChannels, a.chunk};
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
  const int ldx = a.ldx, ldw = a.ldw;
  auto load_offset = [&](int rows, int i, int ld) __attribute__((always_inline)) {
    const int r = rows * wave + 8 * i + (lane >> 3);
    return r * ld + (((lane & 7) ^ p_swz(r)) * 16) - 1024 * (i & 3);
  };
#pragma unroll
  for (int i = 0; i < kMB; i++) xv[i] = load_offset(8 * kMB, i, ldx);
#pragma unroll
  for (int i = 0; i < kNA; i++) wv[i] = load_offset(8 * kNA, i, ldw);
  const uint64_t xp = (uint64_t)(uintptr_t)(a.x + (int64_t)m0 * ldx);
  const uint64_t wp = (uint64_t)(uintptr_t)(a.w + (int64_t)n0 * ldw);
  // Bytes of the tile's rows that exist: what lies past them reads as zero.
  const int x_rows = min(a.seq_len - m0, kTokens), w_rows = min(a.n_out - n0, kChannels);
  const int bytes = a.in / 2;
  // The scales of this wave's rows begin at a block of 16 of them; past the last block they
  // read as zeros, which stand for 2^-127.
  const int x_blocks = (a.seq_len + 15) / 16, w_blocks = (a.n_out + 15) / 16;
  const int x_block = m0 / 16 + kMB * wt, w_block = n0 / 16 + kNA * wc;
  const uint64_t xsp = (uint64_t)(uintptr_t)(a.x_scale + 256 * (int64_t)x_block);
  const uint64_t wsp = (uint64_t)(uintptr_t)(a.w_scale + 256 * (int64_t)w_block);
  Scalars s;
  s.x_lo = uniform((uint32_t)xp), s.x_hi = uniform((uint32_t)(xp >> 32));
  s.w_lo = uniform((uint32_t)wp), s.w_hi = uniform((uint32_t)(wp >> 32));
  s.x_rec = uniform((uint32_t)((x_rows - 1) * ldx + bytes));
  s.w_rec = uniform((uint32_t)((w_rows - 1) * ldw + bytes));
  s.steps = uniform((uint32_t)(bytes / kStep));
  s.m0w = uniform(lds_base + 1024u * kNA * wave);
  s.m0x = uniform(lds_base + 1024u * kMB * wave);
  s.xs_lo = uniform((uint32_t)xsp), s.xs_hi = uniform((uint32_t)(xsp >> 32));
  s.ws_lo = uniform((uint32_t)wsp), s.ws_hi = uniform((uint32_t)(wsp >> 32));
  s.xs_rec = uniform(256u * (uint32_t)max(x_blocks - x_block, 0));
  s.ws_rec = uniform(256u * (uint32_t)max(w_blocks - w_block, 0));
  s.xs_step = uniform(256u * (uint32_t)x_blocks);
  s.ws_step = uniform(256u * (uint32_t)w_blocks);
  s.pairs = uniform((s.steps + 1) / 2);
  const int sv = 4 * lane;
  f32x32 c[kAccs<kNA, kMB>];
  S::reduce(c, ra, rb, xv, wv, &sv, s);

  // The lane again, from the lane counter: kept from before the loop it would
  // be spilled across it.
  int lane2;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane2));
  auto sums = [&](int na, int mb) __attribute__((always_inline)) {
    return block_sums<kNA, kMB>(c, na, mb);
  };
  finish_tile<kNA, kMB, S::kLds, kWaves, kMode, kHl, kPlain, kOut>(a, a.n_out, lds, sums, wave,
                                                                   lane2, m0, n0);
}

// The kernel's arguments with the launch order of a shape's tiles, and the grid that runs it.
template <int kNA, int kMB>
ProjMx4Packed pack_args(const ProjMx4Args& a, bool out, dim3& grid) {
  const ProjGrid g = proj_mx4_grid(a.out.seq_len, a.n_total, 32 * kMB, 32 * kNA);
  grid = dim3(kOrderXcds * g.longest);
  ProjMx4Packed p{};
  p.x = a.x, p.w = a.w, p.x_scale = a.x_scale, p.w_scale = a.w_scale;
  p.q_out = a.out.q_out, p.k_out = a.out.k_out;
  if (out) p.ldo = a.out.ldo;
  else p.v_out = a.out.v_out;
  p.q_gamma = a.out.q_gamma, p.k_gamma = a.out.k_gamma, p.table = a.out.table;
  p.ldx = (int32_t)a.ldx, p.ldw = (int32_t)a.ldw;      // below 2^23: check_operands()
  p.in = a.in, p.n_out = a.n_total;
  p.seq_len = a.out.seq_len, p.seq_pad = a.out.seq_pad, p.heads = a.out.heads;
  p.tiles_m = g.order.tiles_m, p.chunk = g.order.chunk, p.eps = a.out.eps;
  return p;
}

inline int too_large(const ProjMx4Args& a) {
  set_error("too many rows or channels for one launch (%d x %d)", a.out.seq_len, a.n_total);
  return H3HIP_EINVAL;
}

}  // namespace

}  // namespace h3hip
