// Rows of bf16 rounded to microscaled 4-bit floats, what the 4-bit projections (proj_mx4.hip)
// multiply, and back. No counterpart in the reference, whose projections are bf16 matmuls
// (Sources/H3Modules/DiTBlock.swift:336-359). The format is MXFP4 of the OCP Microscaling
// Formats specification, v1.0:
//
//   a = max |x| of 32 consecutive values, e = max(floor(log2 a) - 2, -127),
//   q = x / 2^e rounded to e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6), ties to the even code, at most 6
//
// The block's scale is the byte e + 127. 2^e is a power of two and e2m1 has two significant
// bits, so nothing rounds but q: gfx950's conversion of a scaled pair does exactly this.
//
// Scales lie as the projections read them, four bytes to a lane: the byte of row r and block
// b is at [b / 16][r / 16][16 (b % 4) + r % 16][b / 4 % 4]. 16 rows x 512 values are 256
// consecutive bytes, and the unit of work here: a workgroup reads them 16 bytes a lane, 4
// lanes a block, and collects their scales in LDS.
//
// Bound by HBM: 2 bytes read and 17/32 written an element, and the other way round: 31,885 x 5,120,
// x in no cache, 74 us to 4 bits (5.6 TB/s) and 75 back. Workgroups take units in the order of memory;
// down the columns first they took 82.6 and 86, two units a workgroup 78. 637 x 1,001 is a launch and
// two latencies, 4.0 us.
#include <algorithm>
#include <climits>

#include "mx4_block.h"

namespace h3hip {

namespace {

constexpr int kThreads = 256;
constexpr int kUnitRows = 16, kUnitCols = 512;

struct QuantMx4Args {
  const uint16_t* __restrict__ x;
  uint8_t* __restrict__ q;
  uint8_t* __restrict__ scale;
  int64_t ldx, ldq;
  int32_t rows, cols, cols_pad, across, group0;   // units of a row; the launch's first group of rows
};

__global__ __launch_bounds__(kThreads) void quant_mx4_kernel(QuantMx4Args a) {
  __shared__ uint32_t scales[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Units in the order of memory: a row's one after another.
  const int group = (int)(blockIdx.x / (uint32_t)a.across), slab = (int)blockIdx.x - group * a.across;
  const int64_t r0 = kUnitRows * (int64_t)(a.group0 + group);
  const int64_t k = (int64_t)kUnitCols * slab + 8 * lane;
  const int b = lane >> 2;                   // the lane's block of the unit
  u32x4 v[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {              // rows wave, wave + 4, ...
    const int64_t r = r0 + wave + 4 * i;
    v[i] = r < a.rows ? load_bf16x8(a.x + r * a.ldx, k, a.cols) : u32x4{0u, 0u, 0u, 0u};
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int row = wave + 4 * i;
    uint32_t byte;
    const uint32_t codes = mx4_codes(v[i], byte);
    if (r0 + row < a.rows && k < a.cols_pad)
      *reinterpret_cast<uint32_t*>(a.q + (r0 + row) * a.ldq + k / 2) = codes;
    if ((lane & 3) == 0)
      reinterpret_cast<uint8_t*>(scales)[4 * (16 * (b & 3) + row) + (b >> 2)] = (uint8_t)byte;
  }
  __syncthreads();
  if (wave == 0) {
    const int64_t blocks = ((int64_t)a.rows + kUnitRows - 1) / kUnitRows;
    reinterpret_cast<uint32_t*>(a.scale)[64 * (blocks * slab + r0 / kUnitRows) + lane] =
        scales[lane];
  }
}

struct DequantMx4Args {
  const uint8_t* __restrict__ q;
  const uint8_t* __restrict__ scale;
  uint16_t* __restrict__ x;
  int64_t ldq, ldx;
  int32_t rows, cols, across, group0;
};

__global__ __launch_bounds__(kThreads) void dequant_mx4_kernel(DequantMx4Args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Units in the order of memory: a row's one after another.
  const int group = (int)(blockIdx.x / (uint32_t)a.across), slab = (int)blockIdx.x - group * a.across;
  const int64_t r0 = kUnitRows * (int64_t)(a.group0 + group);
  const int64_t k = (int64_t)kUnitCols * slab + 8 * lane;
  const int64_t blocks = ((int64_t)a.rows + kUnitRows - 1) / kUnitRows;
  const uint8_t* scales = a.scale + 256 * (blocks * slab + r0 / kUnitRows);
  const int b = lane >> 2;
  if (k >= a.cols) return;
  uint32_t codes[4], bytes[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int row = wave + 4 * i;
    const bool in = r0 + row < a.rows;
    codes[i] = in ? *reinterpret_cast<const uint32_t*>(a.q + (r0 + row) * a.ldq + k / 2) : 0u;
    bytes[i] = in ? scales[4 * (16 * (b & 3) + row) + (b >> 2)] : 0u;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t r = r0 + wave + 4 * i;
    if (r >= a.rows) continue;
    const float s = mx4_scale(bytes[i]);
    u32x4 v;
    v[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], s, 0));
    v[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], s, 1));
    v[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], s, 2));
    v[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[i], s, 3));
    if (bytes[i] == kMx4NanScale) v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    uint16_t* dst = a.x + r * a.ldx + k;
    if (k + 8 <= a.cols) {
      *reinterpret_cast<u32x4_any*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k + e < a.cols) dst[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
    }
  }
}

// A launch takes fewer than 2^32 threads.
constexpr int64_t kMaxUnits = (int64_t)1 << 23;
constexpr int32_t kMaxCols = 65535 * kUnitCols;

bool aligned(const void* p, uintptr_t to) {
  return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0;
}

// launch(first group of rows, workgroups) until all of them are through.
template <class Launch>
void for_all_groups(int32_t rows, int across, const Launch& launch) {
  const int64_t groups = ((int64_t)rows + kUnitRows - 1) / kUnitRows;
  const int64_t at_once = kMaxUnits / across;
  for (int64_t g = 0; g < groups; g += at_once)
    launch((int32_t)g, (unsigned)(std::min(groups - g, at_once) * across));
}

}  // namespace

}  // namespace h3hip

using namespace h3hip;

extern "C" int h3hip_quant_rows_mx4(const void* x, int64_t ldx, int32_t rows, int32_t cols, void* q,
                                    int64_t ldq, void* scale, void* stream) {
  H3_REQUIRE(rows >= 0 && cols > 0 && cols <= kMaxCols, H3HIP_EINVAL, "bad shape: rows %d cols %d",
             rows, cols);
  const int cols_pad = (cols + 255) / 256 * 256;
  H3_REQUIRE(ldx >= cols && ldq >= cols_pad / 2 && ldq % 16 == 0, H3HIP_EINVAL,
             "ldx %lld must cover a row, ldq %lld the bytes of the row padded to %d and be a "
             "multiple of 16", (long long)ldx, (long long)ldq, cols_pad);
  if (rows == 0) return H3HIP_OK;
  H3_REQUIRE(x && q && scale, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(aligned(x, 2) && aligned(q, 16) && aligned(scale, 4), H3HIP_EINVAL,
             "x must be 2-byte, q 16-byte and scale 4-byte aligned");
  const int across = (cols_pad + kUnitCols - 1) / kUnitCols;
  for_all_groups(rows, across, [&](int32_t group0, unsigned grid) {
    quant_mx4_kernel<<<dim3(grid), kThreads, 0, as_stream(stream)>>>(
        QuantMx4Args{static_cast<const uint16_t*>(x), static_cast<uint8_t*>(q),
                     static_cast<uint8_t*>(scale), ldx, ldq, rows, cols, cols_pad, across, group0});
  });
  return check_launch("quant_mx4_kernel");
}

extern "C" int h3hip_dequant_rows_mx4(const void* q, int64_t ldq, const void* scale, int32_t rows,
                                      int32_t cols, void* x, int64_t ldx, void* stream) {
  H3_REQUIRE(rows >= 0 && cols > 0 && cols <= kMaxCols, H3HIP_EINVAL, "bad shape: rows %d cols %d",
             rows, cols);
  H3_REQUIRE(ldx >= cols && ldq >= (cols + 7) / 8 * 4 && ldq % 4 == 0, H3HIP_EINVAL,
             "ldx %lld must cover a row, ldq %lld a row's bytes and be a multiple of 4",
             (long long)ldx, (long long)ldq);
  if (rows == 0) return H3HIP_OK;
  H3_REQUIRE(q && scale && x, H3HIP_EINVAL, "NULL tensor argument");
  H3_REQUIRE(aligned(x, 2) && aligned(q, 4), H3HIP_EINVAL, "x must be 2-byte, q 4-byte aligned");
  const int across = (cols + kUnitCols - 1) / kUnitCols;
  for_all_groups(rows, across, [&](int32_t group0, unsigned grid) {
    dequant_mx4_kernel<<<dim3(grid), kThreads, 0, as_stream(stream)>>>(
        DequantMx4Args{static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale),
                       static_cast<uint16_t*>(x), ldq, ldx, rows, cols, across, group0});
  });
  return check_launch("dequant_mx4_kernel");
}
