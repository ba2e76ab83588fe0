// Products of 9 to 128 rows with a large weight (gemm_thin.cu).
#pragma once
#include <cuda_runtime.h>

namespace dragon {

constexpr int THIN_MAX_ROWS = 128;

// out[N, M] = X[N, K] W0[K, M], or act(X W0) * (X W1) with the pre-activations in G and U when G is not null.
struct ThinCall {
  const float* X; const float* W0; const float* W1;
  float* out; float* G; float* U;
  float* work;              // thin_work_floats of scratch
  int N, M, K, act;
  int early;                // X is written by the launch before, a dependent of which this one may be
};
long long thin_work_floats(int N, int M, int K, int mats);
int thin_product(const ThinCall& c, cudaStream_t st);

}  // namespace dragon
