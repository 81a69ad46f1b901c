// Launches of the 4-bit QKV projection in H3HIP_ROUND_ONCE: the kernel of proj_mx4_kernel.h with
// the epilogue that keeps the product in fp32 up to the store of Q and K.
#include "proj_mx4_kernel.h"

namespace h3hip {

namespace {

template <int kNA, int kMB, bool kPair>
int launch(const ProjMx4Args& a, hipStream_t st) {
  dim3 grid;
  const ProjMx4Packed p = pack_args<kNA, kMB>(a, false, grid);
  constexpr int kOnce = H3HIP_ROUND_ONCE;
  if (a.out.rot == 128)
    proj_mx4_gemm_kernel<kNA, kMB, kPair, kOnce, 8, false, false><<<grid, kThreads, 0, st>>>(p);
  else
    proj_mx4_gemm_kernel<kNA, kMB, kPair, kOnce, 6, false, false><<<grid, kThreads, 0, st>>>(p);
  return check_launch("proj_mx4_gemm_kernel");
}

}  // namespace

int launch_proj_mx4_once(const ProjMx4Args& a, ProjMx4Tile tile, hipStream_t stream) {
  switch (tile) {
    case ProjMx4Tile::k256x256: return launch<8, 8, false>(a, stream);
    case ProjMx4Tile::k256x224: return launch<8, 7, false>(a, stream);
    case ProjMx4Tile::k256x192: return launch<8, 6, false>(a, stream);
    case ProjMx4Tile::k256x160: return launch<8, 5, false>(a, stream);
    case ProjMx4Tile::k256x128: return launch<8, 4, false>(a, stream);
    case ProjMx4Tile::k128x192: return launch<4, 6, false>(a, stream);
    case ProjMx4Tile::k128x160: return launch<4, 5, false>(a, stream);
    case ProjMx4Tile::k128x128: return launch<4, 4, false>(a, stream);
    case ProjMx4Tile::k128x128p: return launch<4, 4, true>(a, stream);
    case ProjMx4Tile::k128x64p: return launch<4, 2, true>(a, stream);
    case ProjMx4Tile::k128x32p: return launch<4, 1, true>(a, stream);
    default: break;   // no shape fits, or one of part heads, which is never picked
  }
  return too_large(a);
}

}  // namespace h3hip
