// Global norm of many gradient tensors, and clipping:  norm = sqrt(sum over all tensors of g^2),
// g' = g * min(1, max_norm / norm).
//
// Bound by memory: one read of every gradient for the norm, one read and one write where the limit is exceeded.  The
// squares are exact in 64 bits and summed there: 10^9 gradients of any magnitude lose nothing and overflow nothing.
// The tensors are cut into chunks; a fixed number of thread blocks walks the chunk list with a fixed stride, each block
// leaves one partial sum, and the second kernel adds the partial sums in order, so the norm does not vary from run to
// run.  The second kernel goes through the chunks backwards: what the first one read last is still in L2.
// Addresses and sizes travel as launch parameters: nothing is copied to the device and nothing is retained.
#include <cmath>

#include "cu32_host.h"

namespace dragon {
namespace {

constexpr int THREADS = 256;
constexpr long long CHUNK = 8192;         // floats: 8 vectors per thread
constexpr int BLOCKS_PER_SM = 4;

// The tensors of one launch; first[t] = chunks before tensor t.
template <int CAP>
struct TensorList {
  const float* src[CAP];
  float* dst[CAP];
  long long size[CAP];
  int first[CAP + 1];
  int count;
  int in_place;           // every tensor's destination is its source
};

template <int CAP>
__device__ __forceinline__ int tensor_of(const TensorList<CAP>& list, int chunk) {
  int lo = 0, hi = list.count - 1;        // the last tensor whose first chunk is <= chunk (empty tensors have none)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double square(float x) { return static_cast<double>(x) * static_cast<double>(x); }

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) s += part[w];
  return s;
}

// partial[blockIdx.x] = sum of squares of this block's chunks
template <int CAP>
__global__ void __launch_bounds__(THREADS) grad_norm_kernel(const __grid_constant__ TensorList<CAP> list, double* partial) {
  const int chunks = list.first[list.count];
  double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = tensor_of(list, c);
    const long long at = static_cast<long long>(c - list.first[t]) * CHUNK;
    const float* g = list.src[t] + at;
    const int n = static_cast<int>(min(CHUNK, list.size[t] - at));
    // up to three elements before the first 16-byte boundary, then vectors, then up to three behind
    const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) >> 2);
    const int vecs = (n - head) >> 2;
    const float4* gv = reinterpret_cast<const float4*>(g + head);
#pragma unroll
    for (int i = 0; i < CHUNK / 4 / THREADS; ++i) {
      const int v = i * THREADS + threadIdx.x;
      if (v < vecs) {
        const float4 x = __ldg(gv + v);
        s0 += square(x.x); s1 += square(x.y); s2 += square(x.z); s3 += square(x.w);
      }
    }
    const int tail = head + vecs * 4;
    const int edge = static_cast<int>(threadIdx.x);
    if (edge < head) s0 += square(g[edge]);
    if (edge < n - tail) s1 += square(g[tail + edge]);
  }
  const double s = block_sum((s0 + s1) + (s2 + s3));
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// result = {norm, factor}; dst = src * factor.  Where the factor is 1 and a tensor stays in place, nothing is touched.
// A norm that is not finite leaves every element as it is (factor 1): the caller sees it in result[0].
template <int CAP>
__global__ void __launch_bounds__(THREADS) grad_clip_kernel(const __grid_constant__ TensorList<CAP> list,
                                                            const double* partial, int partials, double max_norm,
                                                            float* result, int write_result) {
  double s = 0.0;
  for (int i = threadIdx.x; i < partials; i += THREADS) s += partial[i];
  const double norm = sqrt(block_sum(s));
  const bool clip = norm > max_norm && norm < INFINITY;
  const float factor = clip ? static_cast<float>(max_norm / norm) : 1.0f;
  if (write_result && blockIdx.x == 0 && threadIdx.x == 0) {
    result[0] = static_cast<float>(norm);
    result[1] = factor;
  }
  if (!clip && list.in_place) return;
  const int chunks = list.first[list.count];
  for (int c = chunks - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const int t = tensor_of(list, c);
    const long long at = static_cast<long long>(c - list.first[t]) * CHUNK;
    const float* g = list.src[t] + at;
    float* out = list.dst[t] + at;
    if (!clip && out == g) continue;
    const int n = static_cast<int>(min(CHUNK, list.size[t] - at));
    if (((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
      const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) >> 2);
      const int vecs = (n - head) >> 2;
      const float4* gv = reinterpret_cast<const float4*>(g + head);
      float4* ov = reinterpret_cast<float4*>(out + head);
      // all loads before the first store: source and destination may be the same, so the compiler cannot reorder them
      float4 x[CHUNK / 4 / THREADS];
#pragma unroll
      for (int i = 0; i < CHUNK / 4 / THREADS; ++i) {
        const int v = i * THREADS + threadIdx.x;
        if (v < vecs) x[i] = gv[v];
      }
#pragma unroll
      for (int i = 0; i < CHUNK / 4 / THREADS; ++i) {
        const int v = i * THREADS + threadIdx.x;
        if (v < vecs) {
          if (clip) { x[i].x *= factor; x[i].y *= factor; x[i].z *= factor; x[i].w *= factor; }   // a copy keeps every bit
          ov[v] = x[i];
        }
      }
      const int tail = head + vecs * 4;
      const int edge = static_cast<int>(threadIdx.x);
      if (edge < head) out[edge] = clip ? g[edge] * factor : g[edge];
      if (edge < n - tail) out[tail + edge] = clip ? g[tail + edge] * factor : g[tail + edge];
    } else {      // source and destination never share a 16-byte boundary
      for (int i = threadIdx.x; i < n; i += THREADS) out[i] = clip ? g[i] * factor : g[i];
    }
  }
}

int norm_blocks(long long chunks) {
  const long long most = static_cast<long long>(device_sm_count()) * BLOCKS_PER_SM;
  return static_cast<int>(chunks < 1 ? 1 : chunks < most ? chunks : most);
}

// Fills a list from tensors [from, count) until it is full; returns where it stopped.  Chunks of one launch stay
// below 2^31: a tensor holds at most 2^40 floats.
template <int CAP>
int fill_list(TensorList<CAP>* list, const int64_t* src, const int64_t* dst, const int64_t* sizes, int from, int count) {
  list->count = 0;
  list->first[0] = 0;
  list->in_place = 1;
  int i = from;
  for (; i < count && list->count < CAP; ++i) {
    if (sizes[i] == 0) continue;
    const long long chunks = (sizes[i] + CHUNK - 1) / CHUNK;
    if (list->first[list->count] + chunks >= (1LL << 31)) break;
    const int t = list->count++;
    list->src[t] = reinterpret_cast<const float*>(static_cast<intptr_t>(src[i]));
    list->dst[t] = dst ? reinterpret_cast<float*>(static_cast<intptr_t>(dst[i])) : nullptr;
    if (!dst || dst[i] != src[i]) list->in_place = 0;
    list->size[t] = sizes[i];
    list->first[t + 1] = list->first[t] + static_cast<int>(chunks);
  }
  return i;
}

template <int CAP>
int clip_all(cudaStream_t st, const int64_t* src, const int64_t* dst, const int64_t* sizes, int count, double max_norm,
             float* result, double* work, long long work_doubles, bool scale) {
  TensorList<CAP> list;
  int partials = 0;
  for (int from = 0; from < count;) {
    from = fill_list(&list, src, dst, sizes, from, count);
    if (list.count == 0) break;
    const int blocks = norm_blocks(list.first[list.count]);
    if (partials + blocks > work_doubles) return CU32_E_SCRATCH;
    grad_norm_kernel<CAP><<<blocks, THREADS, 0, st>>>(list, work + partials);
    if (cudaError_t e = cudaPeekAtLastError()) return static_cast<int>(e);
    partials += blocks;
  }
  bool first = true;
  if (scale)
    for (int from = 0; from < count;) {
      from = fill_list(&list, src, dst, sizes, from, count);
      if (list.count == 0) break;
      const int blocks = norm_blocks(list.first[list.count]);
      grad_clip_kernel<CAP><<<blocks, THREADS, 0, st>>>(list, work, partials, max_norm, result, first ? 1 : 0);
      if (cudaError_t e = cudaPeekAtLastError()) return static_cast<int>(e);
      first = false;
    }
  if (first) {       // the norm alone, or nothing but empty tensors
    list.count = 0;
    list.first[0] = 0;
    grad_clip_kernel<CAP><<<1, THREADS, 0, st>>>(list, work, partials, max_norm, result, 1);
  }
  return static_cast<int>(cudaPeekAtLastError());
}

int grad_any(int64_t stream, const int64_t* src, const int64_t* dst, const int64_t* sizes, int count, float max_norm,
             float* result, double* work, long long work_doubles, bool scale) {
  if (!src || !sizes || (scale && !dst) || !result || !work) return CU32_E_NULL;
  if (count <= 0) return CU32_E_DIM;
  if (!(max_norm >= 0.0f)) return CU32_E_ARG;
  if ((reinterpret_cast<uintptr_t>(work) & 7) || (reinterpret_cast<uintptr_t>(result) & 3)) return CU32_E_ALIGN;
  if (work_doubles < cu32_gradClip_work(count)) return CU32_E_SCRATCH;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0 || sizes[i] > (1LL << 40)) return CU32_E_DIM;
    if (sizes[i] == 0) continue;
    if (!src[i] || (scale && !dst[i])) return CU32_E_NULL;
    if ((src[i] & 3) || (scale && (dst[i] & 3))) return CU32_E_ALIGN;
  }
  const cudaStream_t st = as_stream(stream);
  const double limit = static_cast<double>(max_norm);
  if (count <= 64) return clip_all<64>(st, src, dst, sizes, count, limit, result, work, work_doubles, scale);
  return clip_all<1000>(st, src, dst, sizes, count, limit, result, work, work_doubles, scale);
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

long long cu32_gradClip_work(int count) {
  // a launch holds 1000 tensors and leaves at most BLOCKS_PER_SM partial sums per SM
  if (count <= 0) return 0;
  return static_cast<long long>((count + 999) / 1000 + 1) * device_sm_count() * BLOCKS_PER_SM;
}
int cu32_gradNorm(int64_t stream, const int64_t* src, const int64_t* sizes, int count, float* result, double* work,
                  long long work_doubles) {
  return grad_any(stream, src, nullptr, sizes, count, INFINITY, result, work, work_doubles, false);
}
int cu32_gradClip(int64_t stream, const int64_t* src, const int64_t* dst, const int64_t* sizes, int count, float max_norm,
                  float* result, double* work, long long work_doubles) {
  return grad_any(stream, src, dst, sizes, count, max_norm, result, work, work_doubles, true);
}

}  // extern "C"
