// Launches of the int8 projections' kernel (proj_i8_kernel.h): a tile shape by size
// (proj_i8_tile.h), in the forms of the out-projection, the plain QKV product and the QKV
// product with norm and rotation in two roundings (the third: proj_i8_once.hip).
#include "proj_i8_kernel.h"

namespace h3hip {

namespace {

template <int kNA, int kMB, bool kPair>
int launch(ProjI8Args a, int32_t rounding, bool plain, bool out, hipStream_t st) {
  const dim3 grid = order_grid<kNA, kMB>(a);
  constexpr int kRef = H3HIP_ROUND_REFERENCE, kF32 = H3HIP_ROUND_FP32;
  if (out) {
    proj_i8_gemm_kernel<kNA, kMB, kPair, kRef, 8, true, true><<<grid, kThreads, 0, st>>>(a);
  } else if constexpr (kNA >= 4) {
    if (plain)
      proj_i8_gemm_kernel<kNA, kMB, kPair, kRef, 8, true, false><<<grid, kThreads, 0, st>>>(a);
    else if (rounding == kRef && a.out.rot == 128)
      proj_i8_gemm_kernel<kNA, kMB, kPair, kRef, 8, false, false><<<grid, kThreads, 0, st>>>(a);
    else if (rounding == kRef)
      proj_i8_gemm_kernel<kNA, kMB, kPair, kRef, 6, false, false><<<grid, kThreads, 0, st>>>(a);
    else if (a.out.rot == 128)
      proj_i8_gemm_kernel<kNA, kMB, kPair, kF32, 8, false, false><<<grid, kThreads, 0, st>>>(a);
    else
      proj_i8_gemm_kernel<kNA, kMB, kPair, kF32, 6, false, false><<<grid, kThreads, 0, st>>>(a);
  }
  return check_launch("proj_i8_gemm_kernel");
}

}  // namespace

int launch_proj_i8_gemm(const ProjI8Args& a, int32_t rounding, bool plain, bool out,
                        hipStream_t stream) {
  const ProjI8Tile tile = pick_proj_i8_tile(a.out.seq_len, a.n_total, a.in / kStep, !out);
  if (rounding == H3HIP_ROUND_ONCE && !plain) return launch_proj_i8_once(a, tile, stream);
  switch (tile) {
    case ProjI8Tile::k256x256: return launch<8, 8, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k256x224: return launch<8, 7, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k256x192: return launch<8, 6, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k256x160: return launch<8, 5, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k256x128: return launch<8, 4, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x192: return launch<4, 6, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x160: return launch<4, 5, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x128: return launch<4, 4, false>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x128p: return launch<4, 4, true>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x64p: return launch<4, 2, true>(a, rounding, plain, out, stream);
    case ProjI8Tile::k128x32p: return launch<4, 1, true>(a, rounding, plain, out, stream);
    case ProjI8Tile::k64x64p: return launch<2, 2, true>(a, rounding, plain, out, stream);
    case ProjI8Tile::k32x64p: return launch<1, 2, true>(a, rounding, plain, out, stream);
    case ProjI8Tile::k32x32p: return launch<1, 1, true>(a, rounding, plain, out, stream);
    default: break;
  }
  return too_large(a);
}

}  // namespace h3hip
