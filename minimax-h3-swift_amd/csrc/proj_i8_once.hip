// Launches of the int8 QKV projection in H3HIP_ROUND_ONCE: the kernel of proj_i8_kernel.h with
// the epilogue that keeps the product in fp32 up to the store of Q and K.
#include "proj_i8_kernel.h"

namespace h3hip {

namespace {

template <int kNA, int kMB, bool kPair>
int launch(ProjI8Args a, hipStream_t st) {
  const dim3 grid = order_grid<kNA, kMB>(a);
  constexpr int kOnce = H3HIP_ROUND_ONCE;
  if (a.out.rot == 128)
    proj_i8_gemm_kernel<kNA, kMB, kPair, kOnce, 8, false, false><<<grid, kThreads, 0, st>>>(a);
  else
    proj_i8_gemm_kernel<kNA, kMB, kPair, kOnce, 6, false, false><<<grid, kThreads, 0, st>>>(a);
  return check_launch("proj_i8_gemm_kernel");
}

}  // namespace

int launch_proj_i8_once(const ProjI8Args& a, ProjI8Tile tile, hipStream_t stream) {
  switch (tile) {
    case ProjI8Tile::k256x256: return launch<8, 8, false>(a, stream);
    case ProjI8Tile::k256x224: return launch<8, 7, false>(a, stream);
    case ProjI8Tile::k256x192: return launch<8, 6, false>(a, stream);
    case ProjI8Tile::k256x160: return launch<8, 5, false>(a, stream);
    case ProjI8Tile::k256x128: return launch<8, 4, false>(a, stream);
    case ProjI8Tile::k128x192: return launch<4, 6, false>(a, stream);
    case ProjI8Tile::k128x160: return launch<4, 5, false>(a, stream);
    case ProjI8Tile::k128x128: return launch<4, 4, false>(a, stream);
    case ProjI8Tile::k128x128p: return launch<4, 4, true>(a, stream);
    case ProjI8Tile::k128x64p: return launch<4, 2, true>(a, stream);
    case ProjI8Tile::k128x32p: return launch<4, 1, true>(a, stream);
    default: break;   // no shape fits, or one of part heads, which is never picked
  }
  return too_large(a);
}

}  // namespace h3hip
