// The 4-bit projections of one or two bf16 rows: their rounding and the product in one launch.
//
// What bounds it: W's bytes, 17/32 of one a value (5,120 x 5,120: 14 MB, 2.9 us at the rate of a
// large copy), the launch and the latencies in a row of the rows' loads, W's and the store. So
// a workgroup takes 16 channels over the whole reduction (320 workgroups for 5,120) and has all of
// its W in flight (of reductions up to 10,240) before it does anything else; while that
// arrives, its four waves round the rows into LDS, every workgroup all of them (a row of 5,120 is
// 640 lanes' work). A wave takes every fourth 256 values of the reduction: A is 16 rows of W
// straight from memory, B the rows' codes from LDS, in v_mfma_scale_f32_16x16x128_f8f6f4 as in
// proj_mx4_kernel.h. The four sums are added in LDS, in one order.
//
// Of Q | K | V, whose head norm needs 128 channels at once, the fp32 sums go where the head's
// rows behind the tokens end up as zeros, and a second launch of a workgroup a head norms, rotates
// and stores them. One token x 5,120 x 40 heads takes 12.4 us replayed from a graph, 14.0 of a W that
// no cache holds. Workgroups of 16 waves and whole heads, all of W in flight, need one launch and
// leave half the CUs idle, whose loads are what W takes: 14.4 and 17.0 (host included, where the
// second launch counts, 13.9 instead of 15.8); the tiles of 128 x 32 behind a rounding of their
// own take 13.4 and 17.3.
#include <algorithm>

#include "few_mx4.h"
#include "mx4_block.h"
#include "proj_rows.h"

namespace h3hip {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Rows that a call may have. Every workgroup rounds all of them, and a head's sums wait for a second
// launch: against the rounding and the tiles, replayed, with a W in no cache, one row takes 6.6 us and
// 8.4 (5,120 x 5,120), 8.0 and 9.6 (7,168 x 5,376), 14.6 and 17.9 (5,120, 40 heads), 19.0 and 18.8 (5,376,
// 56 heads), two rows 7.9 and 9.3, 9.4 and 9.7, 16.2 and 17.9, 21.9 and 18.8; with W in the caches 5.2 and
// 6.7, 6.3 and 7.5, 12.5 and 13.3, 17.4 and 15.9; 6.2 and 6.9, 7.7 and 7.5, 14.0 and 13.5, 20.3 and 16.0. It
// needs no workspace either, 1.2 us of the host's time. Two rows of 56 heads are where the tiles
// are ahead already: three and more go there.
constexpr int kMaxRows = 2;
constexpr int kWaves = 4, kThreads = 64 * kWaves, kChannels = 16;
constexpr int kUnitBytes = 128;          // 256 values: two products
constexpr int kMaxHold = 10;             // units of a wave in flight
constexpr int kAtOnce = 4;               // of a lane's 8 values in flight while rows are rounded
constexpr int kSumStride = kChannels + 4;

// LDS: the waves' sums, the rows' codes and their scales, with units up to whole batches.
__host__ __device__ inline int padded_units(int units, int hold) {
  return (units + kWaves * hold - 1) / (kWaves * hold) * (kWaves * hold);
}
inline int64_t lds_bytes(int rows, int units, int hold) {
  const int64_t p = padded_units(units, hold);
  return rows * (kWaves * kSumStride * 4 + p * kUnitBytes + 8 * p);
}
constexpr int64_t kMaxLds = 65536;
inline int hold_of(int units) { return std::min((units + kWaves - 1) / kWaves, kMaxHold); }

// The fp32 sums of a head's rows, [rows][128], from its row kMaxRows on: rows that are behind the
// last token (seq_pad is a multiple of 128), which few_heads_kernel clears.
__device__ __forceinline__ float* few_sums(uint16_t* head) {
  static_assert(3 * kMaxRows <= 128, "the sums fit behind the tokens");
  return reinterpret_cast<float*>(head + kMaxRows * 128);
}

// kHold units of a wave in flight; kSums: fp32 sums to the heads instead of bf16 to y.
template <int kHold, bool kSums>
__global__ __launch_bounds__(kThreads) void few_mx4_kernel(FewMx4Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * kChannels, rows = a.rows;
  const int units = padded_units(a.units, kHold);   // in LDS: zeros past the last
  float* sums = reinterpret_cast<float*>(lds);
  uint8_t* codes = lds + kWaves * rows * kSumStride * 4;
  uint8_t* scales = codes + rows * units * kUnitBytes;

  // W of the workgroup's channels (past the last one its copies, which are not stored).
  const int channel = min(n0 + lr, a.n_total - 1);
  const uint8_t* w = a.w + channel * a.ldw + 16 * g;
  const int64_t slab = 256 * (((int64_t)a.n_total + 15) / 16);
  const uint8_t* ws = a.w_scale + 256 * (int64_t)blockIdx.x + 4 * lane;
  u32x4 wv[kHold][2];
  uint32_t sv[kHold];
  // A batch of this wave's units from u0 on; for units past the last its copies, which meet
  // codes of zero and a scale of one. No branch: it would make every load wait for itself.
  auto load_batch = [&](int u0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kHold; i++) {
      const int u = min(u0 + kWaves * i, a.units - 1);
      wv[i][0] = *reinterpret_cast<const u32x4*>(w + (int64_t)u * kUnitBytes);
      wv[i][1] = *reinterpret_cast<const u32x4*>(w + (int64_t)u * kUnitBytes + 64);
      sv[i] = *reinterpret_cast<const uint32_t*>(ws + slab * (u >> 1));
    }
  };

  // The rows to LDS: 8 values a lane, 4 lanes a block; a part is what the workgroup's lanes hold of
  // a row at once. Loads return in order, so the first parts' are issued before W's.
  const int chunks = 32 * units, parts = (chunks + kThreads - 1) / kThreads;
  u32x4 v[kAtOnce];
  auto load_parts = [&](int p0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int p = min(p0 + i, rows * parts - 1), row = p >= parts ? 1 : 0;
      const int col = min(8 * (tid + (p - row * parts) * kThreads), a.cols - 8);
      v[i] = *reinterpret_cast<const u32x4_any*>(a.x + row * a.ldx + col);
    }
  };
  load_parts(0);
  __builtin_amdgcn_sched_barrier(0);
  load_batch(wave);
  __builtin_amdgcn_sched_barrier(0);
  for (int p0 = 0; p0 < rows * parts; p0 += kAtOnce) {
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const int p = p0 + i, row = p >= parts ? 1 : 0, c = tid + (p - row * parts) * kThreads;
      if (8 * c >= a.cols) v[i] = u32x4{0u, 0u, 0u, 0u};
      uint32_t byte;
      const uint32_t q = mx4_codes(v[i], byte);
      if (p < rows * parts && c < chunks) {
        *reinterpret_cast<uint32_t*>(codes + row * units * kUnitBytes + 4 * c) = q;
        if ((c & 3) == 0) scales[row * 8 * units + (c >> 2)] = (uint8_t)byte;
      }
    }
    if (p0 + kAtOnce < rows * parts) load_parts(p0 + kAtOnce);
  }
  // W stays in flight across this barrier, which __syncthreads would wait for.
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");

  const int row = min(lr, rows - 1);       // past the last row its copy, not stored
  const uint8_t* x = codes + row * units * kUnitBytes + 16 * g;
  const uint8_t* xs = scales + row * 8 * units + g;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int u0 = wave; u0 < units; u0 += kWaves * kHold) {
    u32x4 b[kHold][2];
    int bs[kHold][2];
#pragma unroll
    for (int i = 0; i < kHold; i++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int u = u0 + kWaves * i;
        b[i][h] = *reinterpret_cast<const u32x4*>(x + u * kUnitBytes + 64 * h);
        bs[i][h] = xs[8 * u + 4 * h];
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kHold; i++) {
      const int u = u0 + kWaves * i;
      // Its two blocks' scales in the low bytes.
      const int as = u < a.units ? (int)(sv[i] >> (16 * (u & 1))) : 0x7f7f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const u32x4 t = wv[i][h], c = b[i][h];
        const i32x8 av = {(int)t[0], (int)t[1], (int)t[2], (int)t[3], 0, 0, 0, 0};
        const i32x8 bv = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
        acc = h == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 0, as, 0,
                                                                        bs[i][h])
                     : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc, 4, 4, 1, as, 0,
                                                                        bs[i][h]);
      }
    }
    if (u0 + kWaves * kHold < units) load_batch(u0 + kWaves * kHold);
  }
  // acc: channels 4g .. +3 of row lr.
  if (lr < rows)
    *reinterpret_cast<f32x4*>(sums + (wave * rows + lr) * kSumStride + 4 * g) = acc;
  __syncthreads();
  if (tid < rows * kChannels) {
    const int r = tid / kChannels, c = tid % kChannels;
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < kWaves; s++) y += sums[(s * rows + r) * kSumStride + c];
    if (n0 + c < a.n_total) {
      if constexpr (kSums)
        few_sums(head_rows(a, n0 / 128))[128 * r + n0 % 128 + c] = y;
      else
        a.y[r * a.ldy + n0 + c] = (uint16_t)(pack_bf16x2(y, y) & 0xffffu);
    }
  }
}

// What it needs of ProjArgs: a launch of 128 bytes of arguments and more takes the host 0.9 us
// longer.
struct FewHeadsArgs {
  const uint16_t* __restrict__ q_gamma;
  const uint16_t* __restrict__ k_gamma;
  const void* __restrict__ table;
  uint16_t* q_out;
  uint16_t* k_out;
  uint16_t* v_out;
  float eps;
  int32_t seq_len, seq_pad, heads;
};

// The heads of the sums that they hold: a workgroup a head, 8 lanes a row in the prologue's layout,
// and zeros into the rows behind the last. kPlain: no norm and rotation.
template <int kMode, int kHl, bool kPlain>
__global__ __launch_bounds__(kThreads) void few_heads_kernel(FewHeadsArgs o) {
  constexpr bool kFull = kHl == 8;
  const int head = (int)blockIdx.x, part = head / o.heads;
  const int row = (int)threadIdx.x >> 3, j = (int)threadIdx.x & 7;
  const bool pair_lane = kFull || j < kHl;
  const int chunk_a = pair_lane ? j : 2 * kHl + 2 * (j - kHl);
  const int chunk_b = pair_lane ? j + kHl : chunk_a + 1;
  uint16_t* rows = head_rows(o, head);
  if (row < o.seq_len) {
    float v[16];
    const float* src = few_sums(rows) + 128 * row;
#pragma unroll
    for (int h = 0; h < 4; h++) {
      const f32x4 t = *reinterpret_cast<const f32x4*>(src + 8 * (h < 2 ? chunk_a : chunk_b) +
                                                      4 * (h & 1));
#pragma unroll
      for (int i = 0; i < 4; i++) v[4 * h + i] = t[i];
    }
    u32x4 oa = pack8(v), ob = pack8(v + 8);
    if (!kPlain && part < 2) {
      if (kMode != H3HIP_ROUND_ONCE) unpack8(oa, v), unpack8(ob, v + 8);   // of the bf16 product
      float gam[16];
      const uint16_t* gsrc = part == 0 ? o.q_gamma : o.k_gamma;
      unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_a), gam);
      unpack8(*reinterpret_cast<const u32x4*>(gsrc + 8 * chunk_b), gam + 8);
      RopeEntry tab[8] = {};
      if (pair_lane) {
#pragma unroll
        for (int i = 0; i < 8; i++) {      // entry 8j + i of the row: c, -s, s, c
          const int64_t at = ((int64_t)row * 8 * kHl + 8 * j + i) * 4;
          if (kMode == H3HIP_ROUND_REFERENCE) {
            const u32x2 t = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(o.table) + at);
            tab[i] = RopeEntry{bf16_lo(t[0]), bf16_lo(t[1])};
          } else {
            const f32x4 t = *reinterpret_cast<const f32x4*>(static_cast<const float*>(o.table) + at);
            tab[i] = RopeEntry{t[0], t[2]};
          }
        }
      }
      norm_rope<kMode, kFull>(v, gam, pair_lane, tab, o.eps, oa, ob);
    }
    uint16_t* dst = rows + row * 128;
    *reinterpret_cast<u32x4*>(dst + 8 * chunk_a) = oa;
    *reinterpret_cast<u32x4*>(dst + 8 * chunk_b) = ob;
  }
  __syncthreads();                         // the sums are read before zeros take their place
  zero_rows<128, kThreads>(o, (int)threadIdx.x, o.seq_len, 128 * head);
}

template <int kHold>
void launch(const FewMx4Args& a, hipStream_t st) {
  const dim3 grid((unsigned)(((int64_t)a.n_total + kChannels - 1) / kChannels));
  const size_t lds = lds_bytes(a.rows, a.units, kHold);
  if (a.k_out)
    few_mx4_kernel<kHold, true><<<grid, kThreads, lds, st>>>(a);
  else
    few_mx4_kernel<kHold, false><<<grid, kThreads, lds, st>>>(a);
}

}  // namespace

bool few_mx4_takes(int32_t rows, int32_t cols) {
  const int64_t units = ((int64_t)cols + 255) / 256;
  return rows <= kMaxRows && cols % 8 == 0 && units <= kMaxLds / kUnitBytes &&
         lds_bytes(rows, (int)units, hold_of((int)units)) <= kMaxLds;
}

int launch_few_mx4(const FewMx4Args& a, hipStream_t st) {
  switch (hold_of(a.units)) {
    case 1: launch<1>(a, st); break;
    case 2: launch<2>(a, st); break;
    case 3: launch<3>(a, st); break;
    case 4: launch<4>(a, st); break;
    case 5: launch<5>(a, st); break;
    case 6: launch<6>(a, st); break;
    case 7: launch<7>(a, st); break;
    case 8: launch<8>(a, st); break;
    case 9: launch<9>(a, st); break;
    default: launch<kMaxHold>(a, st);
  }
  return check_launch("few_mx4_kernel");
}

int launch_few_heads(const ProjArgs& o, int32_t rounding, bool plain, hipStream_t st) {
  constexpr int kRef = H3HIP_ROUND_REFERENCE, kF32 = H3HIP_ROUND_FP32, kOnce = H3HIP_ROUND_ONCE;
  const dim3 grid((unsigned)(3 * o.heads));
  const bool full = o.rot == 128;
  const FewHeadsArgs a{o.q_gamma, o.k_gamma, o.table,   o.q_out,   o.k_out,
                       o.v_out,   o.eps,     o.seq_len, o.seq_pad, o.heads};
  if (plain)
    few_heads_kernel<kRef, 8, true><<<grid, kThreads, 0, st>>>(a);
  else if (rounding == kRef && full)
    few_heads_kernel<kRef, 8, false><<<grid, kThreads, 0, st>>>(a);
  else if (rounding == kRef)
    few_heads_kernel<kRef, 6, false><<<grid, kThreads, 0, st>>>(a);
  else if (rounding == kF32 && full)
    few_heads_kernel<kF32, 8, false><<<grid, kThreads, 0, st>>>(a);
  else if (rounding == kF32)
    few_heads_kernel<kF32, 6, false><<<grid, kThreads, 0, st>>>(a);
  else if (full)
    few_heads_kernel<kOnce, 8, false><<<grid, kThreads, 0, st>>>(a);
  else
    few_heads_kernel<kOnce, 6, false><<<grid, kThreads, 0, st>>>(a);
  return check_launch("few_heads_kernel");
}

}  // namespace h3hip
