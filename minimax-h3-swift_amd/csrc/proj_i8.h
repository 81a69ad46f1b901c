// Arguments of the int8 projections' kernel (proj_i8_kernel.h) and its launch.
#pragma once

#include "proj.h"
#include "proj_i8_tile.h"

namespace h3hip {

// out holds what the epilogue shares with the bf16 projections (outputs, gammas,
// table, sizes; its operands are unused). Operand rows are int8, strides in bytes.
struct ProjI8Args {
  ProjArgs out;
  const int8_t* __restrict__ x;         // [seq_len, in], row stride ldx
  const int8_t* __restrict__ w;         // [n_total, in], row stride ldw
  const float* __restrict__ x_scale;    // [seq_len]
  const float* __restrict__ w_scale;    // [n_total]
  int64_t ldx, ldw;
  int32_t in, n_total;
};

// Launches proj_i8_gemm_kernel on the tile shape that suits the sizes (proj_i8_gemm.hip).
int launch_proj_i8_gemm(const ProjI8Args& a, int32_t rounding, bool plain, bool out,
                        hipStream_t stream);
// The same for Q | K | V in H3HIP_ROUND_ONCE, on a given shape (proj_i8_once.hip).
int launch_proj_i8_once(const ProjI8Args& a, ProjI8Tile tile, hipStream_t stream);

}  // namespace h3hip
