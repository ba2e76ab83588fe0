// Weight gradients of few rows: out[m, n] = sum over k < K of A[k, m] B[k, n] for up to three pairs in one launch
// (deltaWg = X^T deltaG, deltaWu = X^T deltaU, deltaWd = H^T deltaY; K is the number of rows).
//
// With so few terms the outputs' stores are the time: 4 bytes for 2 K flop.  The contraction kernel pays a launch, a set-up
// and an epilogue per product and pads K to 32; here all three matrices are one grid of plain FP32 tiles (packed
// multiply-adds), whose next block loads while the last one stores.
// Training passes, this against the contraction kernel, where the rest of the pass is the same: one row of 324 / 892 24.6 us
// against 37, 8 rows of 1912 / 2816 71 against 106, 8 of 4096 / 10924 317 against 398, 16 of it 355 against 408, 24 449
// against 452; 32 rows of 1024 / 2732 75 against 88, but of 4096 / 10924 491 against 452: hence OUTER_MAX_ROWS.
// (Blocks of one step: 8 rows of 4096 / 10924 349 us.  A's values doubled in shared memory instead of in registers: the same.)
#include <atomic>

#include "cu32_host.h"
#include "gated_thin.h"

namespace dragon {
namespace {

constexpr int TM = 64, TN = 256, MOST_STEPS = 4, OUTER_THREADS = 256;

struct OuterParams {
  OuterPair pair[3];
  int tiles_n[3], first[4];     // tiles of a pair: first[i] ... first[i + 1], the columns fastest
  int K, steps, behind;         // steps: tiles of TM rows that a block takes one after the other
};

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 both(float x) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void fma_pair(f32x2& acc, f32x2 a, f32x2 b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b)); }
__device__ __forceinline__ float2 unpack(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// A block loads the columns of B it needs once, and those of A for all its steps: after that it only multiplies and stores.
// A warp takes 8 rows of a step (their A values are the same for all lanes), a lane 4 columns in each half.
__global__ void __launch_bounds__(OUTER_THREADS, 2) outer_kernel(const __grid_constant__ OuterParams p) {
  extern __shared__ __align__(16) float4 outer_smem[];
  if (p.behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tile = blockIdx.x, which = tile >= p.first[2] ? 2 : tile >= p.first[1] ? 1 : 0;
  const OuterPair& q = p.pair[which];
  const int t = tile - p.first[which], tn = p.tiles_n[which];
  const int rows = TM * p.steps, va = rows / 4, m0 = t / tn * rows, n0 = t % tn * TN;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float4* const bs = outer_smem;                       // [K][TN / 4]
  float4* const as = outer_smem + p.K * (TN / 4);      // [K][va]
  for (int i = threadIdx.x; i < p.K * (TN / 4); i += OUTER_THREADS) {
    const int k = i / (TN / 4), n = n0 + i % (TN / 4) * 4;
    bs[i] = n < q.N ? *reinterpret_cast<const float4*>(q.B + static_cast<long long>(k) * q.N + n) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int i = threadIdx.x; i < p.K * va; i += OUTER_THREADS) {
    const int k = i / va, m = m0 + (i - k * va) * 4;
    as[i] = m < q.M ? *reinterpret_cast<const float4*>(q.A + static_cast<long long>(k) * q.M + m) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();
  for (int step = 0; step < p.steps && m0 + step * TM < q.M; ++step) {
    f32x2 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0ull;
    const float4* ak = as + step * (TM / 4) + warp * 2;
    const float4* bk = bs + lane;
#pragma unroll 2
    for (int k = 0; k < p.K; ++k, ak += va, bk += TN / 4) {
      const ulonglong2 b0 = *reinterpret_cast<const ulonglong2*>(bk);
      const ulonglong2 b1 = *reinterpret_cast<const ulonglong2*>(bk + 32);
      const float4 a0 = ak[0], a1 = ak[1];
      const float a[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f32x2 x = both(a[i]);
        fma_pair(acc[i][0], x, b0.x);
        fma_pair(acc[i][1], x, b0.y);
        fma_pair(acc[i][2], x, b1.x);
        fma_pair(acc[i][3], x, b1.y);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m0 + step * TM + warp * 8 + i;
      if (m >= q.M) break;
      float* row = q.out + static_cast<long long>(m) * q.N;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = n0 + h * 128 + lane * 4;
        const float2 x = unpack(acc[i][h * 2]), y = unpack(acc[i][h * 2 + 1]);
        if (n < q.N) *reinterpret_cast<float4*>(row + n) = make_float4(x.x, x.y, y.x, y.y);
      }
    }
  }
}

}  // namespace

int outer_products(const OuterPair* pairs, int count, int K, bool behind, cudaStream_t st) {
  OuterParams p{};
  // Several steps per block where that leaves blocks for two rounds of the machine.
  auto blocks = [&](int steps) {
    long long n = 0;
    for (int i = 0; i < count; ++i)
      n += static_cast<long long>((pairs[i].M + TM * steps - 1) / (TM * steps)) * ((pairs[i].N + TN - 1) / TN);
    return n;
  };
  p.steps = MOST_STEPS;
  while (p.steps > 1 && blocks(p.steps) < 4LL * device_sm_count()) p.steps /= 2;
  const int smem = K * (TN + TM * p.steps) * 4;
  static std::atomic<int> ready[64];
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return static_cast<int>(e);
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(outer_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               OUTER_MAX_ROWS * (TN + TM * MOST_STEPS) * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
    ready[dev & 63].store(1, std::memory_order_release);
  }
  for (int i = 0; i < 3; ++i) {
    p.first[i + 1] = p.first[i];
    if (i >= count) continue;
    p.pair[i] = pairs[i];
    p.tiles_n[i] = (pairs[i].N + TN - 1) / TN;
    p.first[i + 1] += (pairs[i].M + TM * p.steps - 1) / (TM * p.steps) * p.tiles_n[i];     // M N < 2^31: fits
  }
  p.K = K;
  p.behind = behind ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.first[3]), 1, 1);
  cfg.blockDim = dim3(OUTER_THREADS, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = behind ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, outer_kernel, p));
}

}  // namespace dragon
