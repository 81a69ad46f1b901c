// Arguments of the 4-bit projections' kernel (proj_mx4_kernel.h) and its launch.
#pragma once

#include "proj.h"
#include "proj_mx4_tile.h"

namespace h3hip {

// out holds what the epilogue shares with the bf16 projections (outputs, gammas,
// table, sizes; its operands are unused). Operand rows are bytes of two values, strides in
// bytes; scales lie as h3hip_quant_rows_mx4 writes them.
struct ProjMx4Args {
  ProjArgs out;
  const uint8_t* __restrict__ x;         // [seq_len, in / 2], row stride ldx
  const uint8_t* __restrict__ w;         // [n_total, in / 2], row stride ldw
  const uint8_t* __restrict__ x_scale;   // [ceil(in / 512)][ceil(seq_len / 16)][64][4]
  const uint8_t* __restrict__ w_scale;   // [ceil(in / 512)][ceil(n_total / 16)][64][4]
  int64_t ldx, ldw;
  int32_t in, n_total;
};

// Launches proj_mx4_gemm_kernel on the tile shape that suits the sizes (proj_mx4_gemm.hip).
int launch_proj_mx4_gemm(const ProjMx4Args& a, int32_t rounding, bool plain, bool out,
                         hipStream_t stream);
// The same for Q | K | V in H3HIP_ROUND_ONCE, on a given shape (proj_mx4_once.hip).
int launch_proj_mx4_once(const ProjMx4Args& a, ProjMx4Tile tile, hipStream_t stream);

}  // namespace h3hip
