// Rows of bf16 rounded to int8 with one scale a row: what the int8 projections
// (proj_i8.hip) multiply. No counterpart in the reference, whose projections are
// bf16 matmuls (Sources/H3Modules/DiTBlock.swift:336-359).
//
//   a = max_k |x[k]|,  q[k] = round_half_even(127 x[k] / a),  s = a / 127
//
// Bound by HBM: 2 bytes read and 1 written an element (31,885 x 5,120 in 92 us, 5.3 TB/s; a copy
// of 2 GiB 4.9), of few rows by the launch (3.5 us). A wave owns a row and
// holds it in registers between the maximum and the rounding (16 elements a lane
// and chunk), so x is read once; rows of more than 8 chunks (8,192 elements) are
// read twice, the second time from the caches.
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
constexpr int kWavesWg = 4;                    // rows of a workgroup
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

// kChunks: chunks of the row, held in registers; 0: any number, read twice.
template <int kChunks>
__global__ __launch_bounds__(64 * kWavesWg) void quant_rows_kernel(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * kWavesWg +
                    __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (m >= a.rows) return;
  const uint16_t* row = a.x + m * a.ldx;
  int8_t* out = a.q + m * a.ldq;
  const int k0 = kLaneElems * lane;
  constexpr int kHeld = kChunks ? kChunks : 4;   // chunks in registers at once
  uint32_t v[kHeld][8];
  uint32_t top2 = 0;
  if constexpr (kChunks != 0) {
#pragma unroll
    for (int c = 0; c < kChunks; c++) load_chunk(row, k0 + c * kChunk, a.cols, v[c]);
#pragma unroll
    for (int c = 0; c < kChunks; c++) top2 = chunk_max(v[c], top2);
  } else {
    for (int64_t k = 0; k < a.cols; k += kHeld * kChunk) {
#pragma unroll
      for (int c = 0; c < kHeld; c++) load_chunk(row, k + k0 + c * kChunk, a.cols, v[c]);
#pragma unroll
      for (int c = 0; c < kHeld; c++) top2 = chunk_max(v[c], top2);
    }
  }
  uint32_t top = max(top2 & 0xffffu, top2 >> 16);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  // A row that holds an infinity or a NaN has no int8 form: its scale is NaN, so
  // that whatever is multiplied with it shows, and its values are zeros.
  const bool finite = top < 0x7f80u;
  const float amax = __uint_as_float(top << 16);
  RowScale r{0.f, 0.f};
  if (finite && top != 0) {
    r.pre = amax < 0x1p-100f ? 0x1p100f : 1.f;
    r.inv = 127.0f / (amax * r.pre);
  }
  if (lane == 0) a.scale[m] = finite ? amax / 127.0f : __uint_as_float(0x7fc00000u);
  if (!finite) {
    for (int64_t k = k0; k < a.cols_pad; k += kChunk)
      *reinterpret_cast<u32x4*>(out + k) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  if constexpr (kChunks != 0) {
#pragma unroll
    for (int c = 0; c < kChunks; c++) store_chunk(out, k0 + c * kChunk, a.cols_pad, v[c], r);
  } else {
    for (int64_t k = 0; k < a.cols_pad; k += kHeld * kChunk) {
#pragma unroll
      for (int c = 0; c < kHeld; c++) load_chunk(row, k + k0 + c * kChunk, a.cols, v[c]);
#pragma unroll
      for (int c = 0; c < kHeld; c++) store_chunk(out, k + k0 + c * kChunk, a.cols_pad, v[c], r);
    }
  }
}

// A launch takes fewer than 2^32 threads.
constexpr int32_t kMaxRows = (1 << 30) / 64;

void launch(const QuantArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.rows + kWavesWg - 1) / kWavesWg));
  const int chunks = (a.cols_pad + kChunk - 1) / kChunk;
  switch (chunks) {
#define H3_CHUNKS(N) \
  case N: quant_rows_kernel<N><<<grid, 64 * kWavesWg, 0, st>>>(a); break
    H3_CHUNKS(1);
    H3_CHUNKS(2);
    H3_CHUNKS(3);
    H3_CHUNKS(4);
    H3_CHUNKS(5);
    H3_CHUNKS(6);
    H3_CHUNKS(7);
    H3_CHUNKS(8);
#undef H3_CHUNKS
    default: quant_rows_kernel<0><<<grid, 64 * kWavesWg, 0, st>>>(a);
  }
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
