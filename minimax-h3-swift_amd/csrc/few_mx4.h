// Arguments of the 4-bit projections of one or two bf16 rows (few_mx4.hip) and their launches.
#pragma once

#include "proj.h"

namespace h3hip {

struct FewMx4Args {
  const uint16_t* __restrict__ x;        // [rows, cols], row stride ldx elements
  const uint8_t* __restrict__ w;         // [n_total, units * 128], row stride ldw bytes
  const uint8_t* __restrict__ w_scale;
  // y [rows, n_total], row stride ldy elements; or, where k_out is not NULL, heads [heads,
  // seq_pad, 128] of Q, K and V, in each of which the sums are left (few_sums()).
  union {
    uint16_t* y;
    uint16_t* q_out;
  };
  uint16_t* k_out;
  uint16_t* v_out;
  int64_t ldx, ldw, ldy;
  int32_t rows, cols, units, n_total;    // units: of 256 values of the reduction
  int32_t heads, seq_pad;
};

// Whether few_mx4_kernel takes a call of these sizes.
bool few_mx4_takes(int32_t rows, int32_t cols);
int launch_few_mx4(const FewMx4Args& a, hipStream_t stream);
// The heads of the sums in them: out as in ProjMx4Args.
int launch_few_heads(const ProjArgs& out, int32_t rounding, bool plain, hipStream_t stream);

}  // namespace h3hip
