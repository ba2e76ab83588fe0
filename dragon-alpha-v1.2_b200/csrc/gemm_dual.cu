// Kernel instantiations for the sum of two products C = A*B^T + A2*B2^T (A[M][K], B[N][K]): one pass over C, the second
// product's k-blocks behind the first's.
#include "gemm_launch.h"

namespace dragon {

cudaError_t launch_gemm_dual(int tile_cfg, const GemmParams& p, int grid_z, cudaStream_t stream) {
  switch (tile_cfg) {
    case TILE_1x64:  return launch_one<GemmCfg<64, 1, false, false, true, false, false, false, EPI_DUAL>>(p, grid_z, stream);
    case TILE_1x128: return launch_one<GemmCfg<128, 1, false, false, true, false, false, false, EPI_DUAL>>(p, grid_z, stream);
    case TILE_2x128: return launch_one<GemmCfg<128, 2, false, false, true, false, false, false, EPI_DUAL>>(p, grid_z, stream);
    case TILE_2x256: return launch_one<GemmCfg<256, 2, false, false, true, false, false, false, EPI_DUAL>>(p, grid_z, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dragon
