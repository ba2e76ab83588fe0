// Products of the gated block with few rows: with a large weight (gemm_thin.cu), and the weights' gradients
// (gated_outer.cu).
#pragma once
#include <cuda_runtime.h>

namespace dragon {

constexpr int THIN_MAX_ROWS = 128;

enum ThinForm {
  THIN_PLAIN,      // out[N, M] = X[N, K] W0[K, M]
  THIN_GATED,      // out = act(X W0) * (X W1), the pre-activations in G and U when G is not null
  THIN_DELTA,      // h[N, M] = X[N, K] W0[M, K]^T; out = h * preU * act'(preG), U = h * act(preG)
  THIN_DUAL,       // out[N, M] = X W0[M, K]^T + X1 W1[M, K]^T
};
struct ThinCall {
  const float* X; const float* X1; const float* W0; const float* W1;
  float* out; float* G; float* U;
  const float* preG; const float* preU;
  float* work;              // thin_work_floats of scratch
  int N, M, K, act;
  int early;                // X is written by the launch before, a dependent of which this one may be
};
long long thin_work_floats(int N, int M, int K, ThinForm form);
int thin_product(const ThinCall& c, ThinForm form, cudaStream_t st);

// out[M, N] = A[K, M]^T B[K, N], M and N multiples of 4
struct OuterPair {
  const float* A; const float* B; float* out;
  int M, N;
};
constexpr int OUTER_MAX_ROWS = 24;
// Up to three of them in one launch; behind: the launch before is of the same call.
int outer_products(const OuterPair* pairs, int count, int K, bool behind, cudaStream_t st);

}  // namespace dragon
