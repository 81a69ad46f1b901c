// Rows of bf16 rounded to int8 with one scale a row: what the int8 projections
// (proj_i8.hip) multiply. No counterpart in the reference, whose projections are
// bf16 matmuls (Sources/H3Modules/DiTBlock.swift:336-359).
//
//   a = max_k |x[k]|,  q[k] = round_half_even(127 x[k] / a),  s = a / 127
//
// Bound by HBM: 2 bytes read and 1 written an element (31,885 x 5,120 in 88-92 us, 5.3-5.6 TB/s; a
// copy of 2 GiB 4.9), of few rows by the launch (2.7 us). A row is held in the registers of the
// wave or the workgroup that owns it between the maximum and the rounding (16 elements a
// lane and chunk), so x is read once; rows of more than 16 chunks (16,384 elements) are read
// twice, the second time from the caches.
//
// The quotient is never divided out. With i = 127 / a rounded to fp32, t = x i is
// within 2^-23 (relative) of 127 x / a. x and a have 8-bit mantissas, so a quotient
// that is no tie is at least 1 / (254 * 255) > 2^-16 (relative) away from every n + 1/2,
// and a tie has at most 8 significant bits. Rounding t to 19 significant bits moves
// it by at most 2^-19: it lands exactly on a tie that it stands for and cannot reach
// one that it does not. Adding 1.5 * 2^23 then rounds half to even, and the sum's low
// byte is q in two's complement.
#include <algorithm>
#include <climits>

#include "common.h"

namespace h3hip {

namespace {

constexpr int kLaneElems = 16;                 // consecutive elements of a lane in a chunk
constexpr int kChunk = 64 * kLaneElems;        // elements of a wave's chunk
constexpr int kWavesWg = 4;                    // of a workgroup: a row each, or one shared
constexpr uint32_t kAbs2 = 0x7fff7fffu;

struct QuantArgs {
  const uint16_t* __restrict__ x;
  int8_t* __restrict__ q;
  float* __restrict__ scale;
  int64_t ldx, ldq;
  int32_t rows, cols, cols_pad;
};

// Two bf16 magnitudes compared as unsigned halves: their order is the bits' order,
// and infinities and NaN lie above every finite one.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}

// A lane's 16 elements from column k on, zeros past cols. Rows may begin anywhere: gfx950
// loads 16 bytes from any address.
__device__ __forceinline__ void load_chunk(const uint16_t* row, int64_t k, int cols, uint32_t (&v)[8]) {
  if (k + kLaneElems <= cols) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const u32x4 w = *reinterpret_cast<const u32x4_any*>(row + k + 8 * h);
#pragma unroll
      for (int i = 0; i < 4; i++) v[4 * h + i] = w[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = 0u;
  if (k >= cols) return;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t lo = k + 2 * i < cols ? row[k + 2 * i] : 0u;
    const uint32_t hi = k + 2 * i + 1 < cols ? row[k + 2 * i + 1] : 0u;
    v[i] = lo | hi << 16;
  }
}

__device__ __forceinline__ uint32_t chunk_max(const uint32_t (&v)[8], uint32_t m) {
#pragma unroll
  for (int i = 0; i < 8; i++) m = max_u16x2(m, v[i] & kAbs2);
  return m;
}

// What a row is rounded with: x * pre * inv. pre is 1 but for rows whose largest
// magnitude is so small that 127 / a would overflow.
struct RowScale {
  float pre, inv;
};

__device__ __forceinline__ uint32_t code(float x, const RowScale& r) {
  const float t = x * r.pre * r.inv;
  const uint32_t b = (__float_as_uint(t) + 16u) & ~31u;   // 19 significant bits
  return __float_as_uint(__uint_as_float(b) + 12582912.0f);
}

// The lane's 16 codes into 16 bytes at k, as far as the padded row goes.
__device__ __forceinline__ void store_chunk(int8_t* row, int64_t k, int cols_pad,
                                            const uint32_t (&v)[8], const RowScale& r) {
  if (k >= cols_pad) return;
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t c0 = code(bf16_lo(v[2 * i]), r), c1 = code(bf16_hi(v[2 * i]), r);
    const uint32_t c2 = code(bf16_lo(v[2 * i + 1]), r), c3 = code(bf16_hi(v[2 * i + 1]), r);
    // Low bytes of c0, c1 and of c2, c3, then both pairs.
    const uint32_t p0 = __builtin_amdgcn_perm(c1, c0, 0x0c0c0400u);
    const uint32_t p1 = __builtin_amdgcn_perm(c3, c2, 0x0c0c0400u);
    o[i] = p0 | p1 << 16;
  }
  *reinterpret_cast<u32x4*>(row + k) = o;
}

// kChunks: chunks of a wave's row, held in registers; 0: any number, read twice. kShared:
// the workgroup's waves share a row, wave w taking its chunks w, w + kWavesWg, ...
template <int kChunks, bool kShared>
__global__ __launch_bounds__(64 * kWavesWg) void quant_rows_kernel(QuantArgs a) {
  __shared__ uint32_t tops[kWavesWg];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t m = kShared ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWavesWg + wave;
  if (m >= a.rows) return;
  constexpr int kStride = kShared ? kWavesWg * kChunk : kChunk;   // from chunk to chunk of a wave
  const uint16_t* row = a.x + m * a.ldx;
  int8_t* out = a.q + m * a.ldq;
  const int k0 = kLaneElems * lane + (kShared ? kChunk * wave : 0);
  constexpr int kHeld = kChunks ? kChunks : 4;   // chunks in registers at once
  uint32_t v[kHeld][8];
  uint32_t top2 = 0;
  if constexpr (kChunks != 0) {
#pragma unroll
    for (int c = 0; c < kChunks; c++) load_chunk(row, k0 + c * kStride, a.cols, v[c]);
#pragma unroll
    for (int c = 0; c < kChunks; c++) top2 = chunk_max(v[c], top2);
  } else {
    for (int64_t k = k0; k < a.cols; k += kHeld * kStride) {
#pragma unroll
      for (int c = 0; c < kHeld; c++) load_chunk(row, k + c * kStride, a.cols, v[c]);
#pragma unroll
      for (int c = 0; c < kHeld; c++) top2 = chunk_max(v[c], top2);
    }
  }
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  if constexpr (kShared) {
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWavesWg; w++) top = max(top, tops[w]);
  }
  // A row that holds an infinity or a NaN has no int8 form: its scale is NaN, so
  // that whatever is multiplied with it shows, and its values are zeros.
  const bool finite = top < 0x7f80u;
  const float amax = __uint_as_float(top << 16);
  RowScale r{0.f, 0.f};
  if (finite && top != 0) {
    r.pre = amax < 0x1p-100f ? 0x1p100f : 1.f;
    r.inv = 127.0f / (amax * r.pre);
  }
  if (lane == 0 && (!kShared || wave == 0))
    a.scale[m] = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
  if (!finite) {
    for (int64_t k = k0; k < a.cols_pad; k += kStride)
      *reinterpret_cast<u32x4*>(out + k) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  if constexpr (kChunks != 0) {
#pragma unroll
    for (int c = 0; c < kChunks; c++) store_chunk(out, k0 + c * kStride, a.cols_pad, v[c], r);
  } else {
    for (int64_t k = k0; k < a.cols_pad; k += kHeld * kStride) {
#pragma unroll
      for (int c = 0; c < kHeld; c++) load_chunk(row, k + c * kStride, a.cols, v[c]);
#pragma unroll
      for (int c = 0; c < kHeld; c++) store_chunk(out, k + c * kStride, a.cols_pad, v[c], r);
    }
  }
}

// A launch takes fewer than 2^32 threads.
constexpr int32_t kMaxRows = (1 << 30) / (64 * kWavesWg);

// A row a wave, or a row a workgroup. Shared, a row's latencies are a fourth each (one row of
// 7,168 4.0 -> 2.8 us, 1,151 rows 8.8 -> 7.3), which is what few rows wait for; many rows need the
// bytes in flight, and four waves with a chunk each hold fewer than four with a row each
// (18,102 rows of 3,000 39 -> 42 us, of 2,048 17 -> 19). From two chunks a wave on sharing costs
// nothing (31,885 x 5,120 90 -> 88 us, 18,102 x 6,000 62 -> 58, 4,000 x 12,000 41 -> 28).
constexpr int kFewRows = 2048;

template <bool kShared>
void launch(const QuantArgs& a, int chunks, hipStream_t st) {
  const dim3 grid((unsigned)(kShared ? a.rows : (a.rows + kWavesWg - 1) / kWavesWg));
  const dim3 block(64 * kWavesWg);
  switch (kShared ? (chunks + kWavesWg - 1) / kWavesWg : chunks) {
    case 1: quant_rows_kernel<1, kShared><<<grid, block, 0, st>>>(a); break;
    case 2: quant_rows_kernel<2, kShared><<<grid, block, 0, st>>>(a); break;
    case 3: quant_rows_kernel<3, kShared><<<grid, block, 0, st>>>(a); break;
    case 4: quant_rows_kernel<4, kShared><<<grid, block, 0, st>>>(a); break;
    default: quant_rows_kernel<0, true><<<grid, block, 0, st>>>(a);   // shared
  }
}

void launch(const QuantArgs& a, hipStream_t st) {
  const int chunks = (a.cols_pad + kChunk - 1) / kChunk;
  if (chunks > kWavesWg || (chunks > 2 && a.rows <= kFewRows))
    launch<true>(a, chunks, st);
  else
    launch<false>(a, chunks, st);
}

}  // namespace

}  // namespace h3hip

using namespace h3hip;

extern "C" int h3hip_quant_rows(const void* x, int64_t ldx, int32_t rows, int32_t cols, void* q,
                                int64_t ldq, float* scale, void* stream) {
  H3_REQUIRE(rows >= 0 && cols > 0 && cols <= INT32_MAX - 2 * kChunk, H3HIP_EINVAL,
             "bad shape: rows %d cols %d", rows, cols);
  const int cols_pad = (cols + 127) / 128 * 128;
  H3_REQUIRE(ldx >= cols && ldq >= cols_pad && ldq % 16 == 0, H3HIP_EINVAL,
             "ldx %lld must cover a row, ldq %lld the row padded to %d and be a multiple of 16",
             (long long)ldx, (long long)ldq, cols_pad);
  if (rows == 0) return H3HIP_OK;
  H3_REQUIRE(x && q && scale, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE((reinterpret_cast<uintptr_t>(x) & 1u) == 0 &&
                 (reinterpret_cast<uintptr_t>(q) & 15u) == 0 &&
                 (reinterpret_cast<uintptr_t>(scale) & 3u) == 0,
             H3HIP_EINVAL, "x must be 2-byte, q 16-byte and scale 4-byte aligned");
  for (int64_t m = 0; m < rows; m += kMaxRows)
    launch(QuantArgs{static_cast<const uint16_t*>(x) + m * ldx, static_cast<int8_t*>(q) + m * ldq,
                     scale + m, ldx, ldq, (int32_t)std::min<int64_t>(rows - m, kMaxRows), cols,
                     cols_pad},
           as_stream(stream));
  return check_launch("quant_rows_kernel");
}
