// Kernel instantiations of the gated feed-forward block's first half: act(A*B) * (A*B2) with A[M][K], B[K][N].
#include "gemm_launch.h"

namespace dragon {

cudaError_t launch_gemm_gated(int tile_cfg, const GemmParams& p, cudaStream_t stream) {
  const int grid_z = 1;
  switch (tile_cfg) {
    case TILE_1x128: return launch_one<GemmCfg<128, 1, false, true, true, false, false, false, EPI_GATED>>(p, grid_z, stream);
    case TILE_2x128: return launch_one<GemmCfg<128, 2, false, true, true, false, false, false, EPI_GATED>>(p, grid_z, stream);
    case TILE_2x256: return launch_one<GemmCfg<256, 2, false, true, true, false, false, false, EPI_GATED>>(p, grid_z, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace dragon
