// What the C-ABI translation units share on the host: argument checks, tensor maps and the plain contraction call.
// Defined in cu32_api.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <cstring>

#include "../../include/dragon_cu32.h"
#include "gemm_launch.h"

namespace dragon {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline cudaStream_t as_stream(int64_t s) { return reinterpret_cast<cudaStream_t>(static_cast<intptr_t>(s)); }

// One contraction, BLAS letters: C[M,N] = A * B over K.
struct GemmCall {
  const float* A; const float* B; float* C; float* Cbuf;
  int M, N, K;              // logical extents of the operands
  int n_store;              // columns of C written (>= N; columns N.. come out 0)
  long long lda, ldb, ldc;  // row pitches in floats
  bool a_mn, b_mn;          // operand stored with its M / N axis contiguous
  int batch; long long sA, sB, sC;
  int gz;                   // split-K slices (1 = none)
  bool x3;                  // FP32-accurate (true) or single-pass TF32
  cudaStream_t stream;
  const float* bias;        // optional row vector (n_store floats) added in the epilogue; needs gz == 1, batch == 1
  int bias_width;           // true width of the rows: columns beyond it are stored as zeros
  bool scale_on = false;   // store alpha * result (one rounding), vector store paths only
  float alpha = 1.0f;
  float* const* replicas = nullptr;   // further output buffers that receive the same stores as C (same layout)
  int n_replicas = 0;
  int kc = 0;                         // k-blocks per in-TMEM chunk; 0 = the "kc" tuning keys
  bool beside_prev = false;           // may run beside the previous launch on the stream, which it does not depend on
  bool behind_prev = false;           // the previous launch on the stream is this call's own: start up beside its end
};

int run_gemm(const GemmCall& c);

// Environment overrides of the tuning integers, read once.
void load_env_once();
// CU32_OK and streams[0], or CU32_E_STREAMS.
int check_streams(const int64_t* streams, int length, cudaStream_t* s0);
// Resolves the driver's tensor-map encoders once; false when they are not available.
bool load_driver_entry_points();
// 3-D FP32 map (inner, outer, batch) with zero fill; see cu32_api.cu for the swizzles.
int make_map3(CUtensorMap* m, const float* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t pitch1_floats,
              uint64_t pitch2_floats, uint32_t b0, uint32_t b1, bool mn_major);
int make_map3_as(CUtensorMap* m, const float* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t pitch1_floats,
                 uint64_t pitch2_floats, uint32_t b0, uint32_t b1, CUtensorMapSwizzle swizzle);
// k-blocks per in-TMEM chunk of the gated block's products.  Their errors add up along the block (G, U, H, Y and back), and
// the tensor core's truncation grows with the chunk: with one the block's results are 6e-7 off, with two (the plain
// products' default) 1.3e-6, for 2 to 5 % of its time.
constexpr int GATED_KC = 1;
// The "tile" tuning key: a forced tile configuration, or -1.
int forced_tile();
// Counts a product that went in two pieces of columns for the "column_cuts" tuning key.
void note_column_cut();
// The "rows_give_up" tuning key.
int rows_give_up();
// Ring lengths, flush interval, clock accumulator and reserved SMs of a launch, from the tuning integers.
void choose_rings(GemmParams* p);
// Give-up word of the current device.
int* status_word_ptr(cudaError_t* err);
// Remembers the tile a call uses for the "last_tile" tuning key.
int note_tile(int t);

}  // namespace dragon
