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
constexpr int VPT = CHUNK / 4 / THREADS;
// The norm's grid is persistent, eight blocks per SM (32 registers a thread; many blocks hide the look-up of a chunk: 228 us
// against 244 with four for 1.6 GB).  The clipping's has a block per chunk where it writes elsewhere, and four rounds of
// blocks in place: blocks that start in order keep what is read and written at one time close together, which persistent
// blocks that drift apart do not (1.6 GB out of place: 491 us against 607 with five blocks per SM).  In place above the limit
// the whole call takes 790 us for 1.6 GB, elsewhere 718; below the limit 12,000 blocks with nothing to do would add 6 us.
constexpr int NORM_BLOCKS_PER_SM = 8, CLIP_BLOCKS_PER_SM = 5;

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

// One chunk: where it lies, and how its n elements fall on 16-byte boundaries - up to three before the first, then
// vectors, then up to three behind.
struct Chunk {
  const float* g;
  float* out;
  int n, head, vecs;
};
template <int CAP>
__device__ __forceinline__ Chunk locate(const TensorList<CAP>& list, int c) {
  const int t = tensor_of(list, c);
  const long long at = static_cast<long long>(c - list.first[t]) * CHUNK;
  Chunk x;
  x.g = list.src[t] + at;
  x.out = list.dst[t] + at;
  x.n = static_cast<int>(min(CHUNK, list.size[t] - at));
  x.head = min(x.n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x.g) & 15)) & 15) >> 2);
  x.vecs = (x.n - x.head) >> 2;
  return x;
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
__global__ void __launch_bounds__(THREADS, NORM_BLOCKS_PER_SM) grad_norm_kernel(const __grid_constant__ TensorList<CAP> list, double* partial) {
  const int chunks = list.first[list.count];
  double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Chunk x = locate(list, c);
    const float4* gv = reinterpret_cast<const float4*>(x.g + x.head);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * THREADS + threadIdx.x;
      if (v < x.vecs) {
        const float4 q = __ldg(gv + v);
        s0 += square(q.x); s1 += square(q.y); s2 += square(q.z); s3 += square(q.w);
      }
    }
    const int tail = x.head + x.vecs * 4, edge = static_cast<int>(threadIdx.x);
    if (edge < x.head) s0 += square(x.g[edge]);
    if (edge < x.n - tail) s1 += square(x.g[tail + edge]);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const double s = block_sum((s0 + s1) + (s2 + s3));
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// Norm and factor from the partial sums, the same in every thread of the block.
__device__ __forceinline__ void norm_of(const double* partial, int partials, double max_norm, double* norm, double* factor) {
  double s = 0.0;
  for (int i = threadIdx.x; i < partials; i += THREADS) s += partial[i];
  *norm = sqrt(block_sum(s));
  *factor = *norm > max_norm && *norm < INFINITY ? max_norm / *norm : 1.0;
}
__device__ __forceinline__ void store_result(double norm, double factor, float* result) {
  result[0] = static_cast<float>(norm);
  result[1] = static_cast<float>(factor);
}
// result = {norm, factor}, and the factor in 64 bits behind the partial sums; one block
__global__ void __launch_bounds__(THREADS) grad_result_kernel(double* partial, int partials, double max_norm, float* result) {
  double norm, factor;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  norm_of(partial, partials, max_norm, &norm, &factor);
  if (threadIdx.x == 0) {
    store_result(norm, factor, result);
    partial[partials] = factor;
  }
}

// Below the smallest normal FP32 number (2^-126) a factor would lose bits, or all of itself: the products are formed in 64
// bits there, element by element (norms above 8.5e37 times the limit: not a case to be fast in).
constexpr double SMALLEST_FACTOR = 1.1754943508222875e-38;

// dst = src * factor.  Where the factor is 1 and a tensor stays in place, nothing is touched.  A norm that is not finite
// leaves every element as it is (factor 1): the caller sees it in result[0].  direct: the blocks form norm and factor
// themselves, and the first one writes the result; else the factor lies behind the partial sums.
template <int CAP>
__global__ void __launch_bounds__(THREADS, CLIP_BLOCKS_PER_SM) grad_clip_kernel(const __grid_constant__ TensorList<CAP> list,
                                                                               const double* partial, int partials, int direct,
                                                                               double max_norm, float* result) {
  double wide;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (direct) {
    double norm;
    norm_of(partial, partials, max_norm, &norm, &wide);
    if (blockIdx.x == 0 && threadIdx.x == 0) store_result(norm, wide, result);
  } else {
    wide = partial[partials];
  }
  const float factor = static_cast<float>(wide);
  const bool clip = factor != 1.0f;
  if (!clip && list.in_place) return;
  const int chunks = list.first[list.count];
  if (wide > 0.0 && wide < SMALLEST_FACTOR) {
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
      const Chunk k = locate(list, c);
      for (int i = threadIdx.x; i < k.n; i += THREADS) k.out[i] = static_cast<float>(static_cast<double>(k.g[i]) * wide);
    }
    return;
  }
  int c = chunks - 1 - static_cast<int>(blockIdx.x);
  Chunk next = c >= 0 ? locate(list, c) : Chunk{};
  for (; c >= 0; c -= gridDim.x) {
    const Chunk k = next;
    const int after = c - static_cast<int>(gridDim.x);
    const bool stays = !clip && k.out == k.g;
    if (stays || ((reinterpret_cast<uintptr_t>(k.g) ^ reinterpret_cast<uintptr_t>(k.out)) & 15) != 0) {
      if (!stays)     // source and destination never share a 16-byte boundary
        for (int i = threadIdx.x; i < k.n; i += THREADS) k.out[i] = clip ? k.g[i] * factor : k.g[i];
      if (after >= 0) next = locate(list, after);
      continue;
    }
    const float4* gv = reinterpret_cast<const float4*>(k.g + k.head);
    float4* ov = reinterpret_cast<float4*>(k.out + k.head);
    // all loads before the first store: source and destination may be the same, so the compiler cannot reorder them
    float4 x[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * THREADS + threadIdx.x;
      if (v < k.vecs) x[i] = gv[v];
    }
    if (after >= 0) next = locate(list, after);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * THREADS + threadIdx.x;
      if (v < k.vecs) {
        if (clip) { x[i].x *= factor; x[i].y *= factor; x[i].z *= factor; x[i].w *= factor; }   // a copy keeps every bit
        ov[v] = x[i];
      }
    }
    const int tail = k.head + k.vecs * 4, edge = static_cast<int>(threadIdx.x);
    if (edge < k.head) k.out[edge] = clip ? k.g[edge] * factor : k.g[edge];
    if (edge < k.n - tail) k.out[tail + edge] = clip ? k.g[tail + edge] * factor : k.g[tail + edge];
  }
}

int blocks_of(long long chunks, int per_sm) {
  const long long most = static_cast<long long>(device_sm_count()) * per_sm;
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

// A launch that waits for the one before it on the device, its start-up beside that one's end.
template <class... P, class... A>
cudaError_t launch_behind(void (*kernel)(P...), int blocks, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int CAP>
int clip_all(cudaStream_t st, const int64_t* src, const int64_t* dst, const int64_t* sizes, int count, double max_norm,
             float* result, double* work, long long work_doubles, bool scale) {
  TensorList<CAP> list;
  int partials = 0, lists = 0;
  for (int from = 0; from < count;) {
    from = fill_list(&list, src, dst, sizes, from, count);
    if (list.count == 0) break;
    const int blocks = blocks_of(list.first[list.count], NORM_BLOCKS_PER_SM);
    if (partials + blocks + 1 > work_doubles) return CU32_E_SCRATCH;
    grad_norm_kernel<CAP><<<blocks, THREADS, 0, st>>>(list, work + partials);
    if (cudaError_t e = cudaPeekAtLastError()) return static_cast<int>(e);
    partials += blocks;
    ++lists;
  }
  // One launch that every block of which can form the norm itself, or the norm first and a block per chunk behind it.
  const bool direct = scale && lists == 1 && list.first[list.count] <= device_sm_count() * CLIP_BLOCKS_PER_SM;
  if (!direct)
    if (cudaError_t e = launch_behind(grad_result_kernel, 1, st, work, partials, max_norm, result))
      return static_cast<int>(e);
  if (!scale || lists == 0) return CU32_OK;
  for (int from = 0; from < count;) {
    if (lists > 1) from = fill_list(&list, src, dst, sizes, from, count);
    else from = count;
    if (list.count == 0) break;
    // in place the blocks may have nothing to do: fewer of them (12,000 that leave at once take 6 us)
    const int blocks = list.in_place ? blocks_of(list.first[list.count], 4 * CLIP_BLOCKS_PER_SM) : list.first[list.count];
    const cudaError_t e = launch_behind(grad_clip_kernel<CAP>, blocks, st, list,
                                        static_cast<const double*>(work), partials, direct ? 1 : 0, max_norm, result);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return CU32_OK;
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
  // a launch holds 1000 tensors and leaves at most NORM_BLOCKS_PER_SM partial sums per SM; one more for the factor
  if (count <= 0) return 0;
  return static_cast<long long>((count + 999) / 1000 + 1) * device_sm_count() * NORM_BLOCKS_PER_SM;
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
