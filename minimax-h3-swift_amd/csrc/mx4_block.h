// A block of 32 bf16 values to MXFP4 on four lanes of 8 values each: shared by the rounding of
// rows (quant_mx4.hip, which states the format) and the projections of few rows (few_mx4.hip).
#pragma once

#include "common.h"

namespace h3hip {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kMx4NanScale = 255u;

__device__ __forceinline__ bf16x2 bf16_pair(uint32_t w) { return __builtin_bit_cast(bf16x2, w); }

// 8 elements from column k on, zeros past cols. Rows may begin anywhere: gfx950 loads 16 bytes
// from any address.
__device__ __forceinline__ u32x4 load_bf16x8(const uint16_t* row, int64_t k, int cols) {
  if (k + 8 <= cols) return *reinterpret_cast<const u32x4_any*>(row + k);
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t lo = k + 2 * i < cols ? row[k + 2 * i] : 0u;
    const uint32_t hi = k + 2 * i + 1 < cols ? row[k + 2 * i + 1] : 0u;
    v[i] = lo | hi << 16;
  }
  return v;
}

// The fp32 2^(byte - 127); 0 is 2^-127, a subnormal.
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 1u << 22 : byte << 23);
}

// The lane's 8 codes, and the block's biased exponent in every lane of it.
__device__ __forceinline__ uint32_t mx4_codes(u32x4 v, uint32_t& byte) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  // Magnitudes of bf16 compare as whole numbers; infinities and NaN lie above the rest.
  u16x2 m = {0, 0};
#pragma unroll
  for (int h = 0; h < 4; h++) {
    const uint32_t w = v[h] & 0x7fff7fffu;
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w));
  }
  uint32_t top = max((uint32_t)m[0], (uint32_t)m[1]);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));
  // A block that holds an infinity or a NaN has no such form: its scale is NaN, so that
  // whatever is multiplied with it shows, and its values are zeros.
  const bool finite = top < 0x7f80u;
  const uint32_t e = top >> 7;             // biased exponent; 0: subnormals and zero
  byte = finite ? (e > 2 ? e - 2 : 0u) : kMx4NanScale;
  const float s = mx4_scale(finite ? byte : 127u);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, bf16_pair(v[0]), s, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, bf16_pair(v[1]), s, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, bf16_pair(v[2]), s, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, bf16_pair(v[3]), s, 3);
  return finite ? codes : 0u;
}

}  // namespace h3hip
