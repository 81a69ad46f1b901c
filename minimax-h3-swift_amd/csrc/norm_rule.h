// How many workgroups of the norms' kernels (norm_residual.hip) are launched a CU. Plain C++, so a
// CPU test can check it against the registers that the kernels compile to.
#pragma once

#include <cstdint>

namespace h3hip {

constexpr int kNormCus = 256;

// Waves a SIMD, to which the compiler is held. One chunk a thread is 6, in 80 registers: in the 94
// that the compiler took by itself two workgroups of 11 waves did not fit a CU (31,885 x 5,376, after
// with a next norm, 373 us; 297). Two chunks hold twice the row and the tables: what their kernels
// need without spilling. after: there is y; post: it is normalised; next: h is written; many: rows of
// more than one segment.
constexpr int norm_waves_simd(int chunks, bool after, bool post, bool next, bool many) {
  if (chunks == 1) return 6;
  if (after && next) return post || many ? 4 : 5;
  if (after) return post && many ? 5 : 6;
  return many ? 4 : 6;
}

// Workgroups a CU of rows of `waves` waves. Below 16 rows a CU as many as fit: a second round of
// them loads the tables again with nothing to cover it (after with a next norm, 300 x 9,000 12.0 us, 9.2
// with as many as fit; 600 x 10,240 13.9 and 11.8; 2,000 x 10,240 34.7 and 33.2). Of more rows as for
// 6 waves a SIMD even where 4 fit: the second round then begins where a CU is done first
// (6,000 x 12,288 120 us, 124 with as many as fit; 18,102 x 10,240 292 and 312, x 9,000 308 and 304).
constexpr int norm_workers_cu(int waves, int rows, int waves_simd) {
  const int simd = rows < 16 * kNormCus ? waves_simd : 6;
  return 4 * simd < waves ? 1 : 4 * simd / waves;
}

}  // namespace h3hip
