// The norms around a block of a residual network, with the block's gate and the residual's scale, in one pass:
//
//   b^ = B / rms(B)            rms(x) = sqrt(mean(x^2) + eps) over the row's `width` columns
//   P  = w_post * b^           (P = B where there is no w_post)
//   R' = res_scale * R + scale * gate * P
//   Y  = w_pre * R' / rms(R')  what the next block reads
//
// and the gradients, from deltaR' (what later layers say about R') and deltaY:
//   q = w_pre deltaY, r^ = R' / rms(R'), c1 = mean(q r^):    dT = deltaR' + (q - r^ c1) / rms(R')
//   deltaR = res_scale dT;  dP = scale gate dT;  deltaGate = sum over its rows of scale P dT
//   c2 = mean(dP w_post b^):  deltaB = (dP w_post - b^ c2) / rms(B)
//   deltaW_pre = sum of deltaY r^;  deltaW_post = sum of dP b^
// c2 needs dT and so c1, which would make two dependent reductions per row; with e = scale gate w_post b^ it is
//   width c2 = sum e (deltaR' + q / rms(R')) - c1 sum e r^ / rms(R'),
// so one reduction of three sums serves the row.
//
// Bound by memory: forward 4 floats per element (B, R in; R', Y out), gradients 6 (four in, two out).  Few rows: a block
// per row, everything at once in its registers.  Many rows: persistent blocks (clusters of two or four for rows of more
// than 4096 columns, each block a part of the row) that keep a ring of rows in shared memory filled by bulk copies: a row
// moves to registers in one step and its place is refilled at once, so that two rows or more are on their way whatever
// the row in hand waits for.  The column sums are kept in registers over all rows of a block, written once per block
// and added in a fixed order by a second, small kernel (no atomics: results do not vary from run to run).
#include <atomic>

#include "cu32_host.h"

namespace dragon {
namespace {

using namespace ptx;

constexpr int MAX_WIDTH = 16384;     // floats per row: a cluster of four blocks of 1024 vectors
// 16-byte vectors per thread of the persistent kernels.  Two, so that the weights fit in the registers beside the sums: a
// ring that fills the shared memory leaves the L1 cache too little for 48 KB of weights, and reading them from L2 for
// every row made the kernels wait for it (with four per thread: 145 us forward, 213 us gradients at 8192 x 4096).
constexpr int VPT = 2;
constexpr int RING_THREADS = 512;
// Holds the gradient kernel to 96 registers (a block has at most RING_THREADS threads; left to itself it takes 118, and one
// block of 288 threads fills an SM instead of two: 8192 x 2052 rows 89 us instead of 79; elsewhere the same).  Of its twelve
// instances one spills, the clusters of two with gate and both norms: 8 bytes stored, 4 read again.
constexpr int DELTA_BOUND = 576;

__device__ __forceinline__ float4 ldg_row(const float* p) {       // read once: not kept in L1
  float4 v;
  asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float4 zero4() { return make_float4(0.f, 0.f, 0.f, 0.f); }
// columns >= width count as 0
__device__ __forceinline__ float4 clip4(float4 v, int col, int width) {
  if (col + 3 >= width) {
    if (col + 0 >= width) v.x = 0.f;
    if (col + 1 >= width) v.y = 0.f;
    if (col + 2 >= width) v.z = 0.f;
    if (col + 3 >= width) v.w = 0.f;
  }
  return v;
}

// On the way out they are 0 as long as the row's factors are finite; else 0 * NaN is put right behind the vector stores, by the
// threads that made them.
__device__ __forceinline__ bool all_finite(float sum_of_factors) { return fabsf(sum_of_factors) <= 3.4e38f; }
__device__ __forceinline__ void clear_padding(float* part, int vec0, int vecs, int width) {
  for (int v = threadIdx.x; v < vecs; v += blockDim.x)
    for (int j = 0; j < 4; ++j)
      if ((vec0 + v) * 4 + j >= width) part[v * 4 + j] = 0.0f;
}

__device__ __forceinline__ float4 ones4() { return make_float4(1.f, 1.f, 1.f, 1.f); }
__device__ __forceinline__ float square_sum(float4 v) { return v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w; }
__device__ __forceinline__ float4 scaled(float4 v, float f, float4 w) {
  return make_float4(v.x * f * w.x, v.y * f * w.y, v.z * f * w.z, v.w * f * w.w);
}
// 1 / sqrt(x): the hardware's estimate and one Newton step (0 and infinity have no step)
__device__ __forceinline__ float inv_root(float x) {
  const float r = rsqrtf(x);
  return x > 0.0f && x < INFINITY ? r * fmaf(-0.5f * x * r, r, 1.5f) : r;
}
// vector v of a row of weights, columns >= width as 0
__device__ __forceinline__ float4 load_weight(const float* w, int v, int width) {
  return clip4(__ldg(reinterpret_cast<const float4*>(w) + v), v * 4, width);
}

// Sum of a value over the threads of the block, the same in every thread.  One barrier per call: the slots alternate, so a
// slot is written again only after everybody has passed the barrier of the call in between.
struct BlockSum {
  float (*slots)[32];     // [2][32]
  int parity = 0;
  __device__ __forceinline__ float operator()(float v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) return v;
    if (lane == 0) slots[parity][warp] = v;
    __syncthreads();
    v = lane < warps ? slots[parity][lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    parity ^= 1;
    return v;
  }
};

// Sums of K values over the warps of a cluster's blocks, the same in every thread; false when a wait ran out.  The slots
// alternate: a slot is written again only after its writer has waited for the set in between, which every warp delivered
// after it had read the slot.
template <int K, int CL>
struct TeamSum {
  float (*slots)[K][64];      // [2][K][64]: by set, value, warp of the cluster (at most 16 per block); zeroed at the start
  uint64_t* bars;             // [2]
  volatile int* abort_flag;
  uint32_t sets = 0;

  __device__ __forceinline__ bool operator()(float (&v)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int par = sets & 1;
    const uint32_t bar = smem_u32(&bars[par]);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (CL == 1) {
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) slots[par][k][warp] = v[k];
        mbar_arrive(bar);
      }
    } else {
      // Lane r delivers to block r; each value carries its own count to that block's barrier.  (An arrival that
      // releases at cluster scope would first wait for this thread's global stores: twice the row's time.)
      if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(warps * CL * K * 4));
      if (lane < CL) {
        const int at = static_cast<int>(cluster_ctarank()) * warps + warp;
        const uint32_t there = mapa(bar, lane);
#pragma unroll
        for (int k = 0; k < K; ++k) st_async(mapa(smem_u32(&slots[par][k][at]), lane), v[k], there);
      }
    }
    if (!mbar_wait(bar, (sets >> 1) & 1u, abort_flag)) return false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float x = slots[par][k][CL == 1 ? lane & 15 : lane];      // both halves of the warp add the same 16
      if (CL > 2) x += slots[par][k][lane + 32];
#pragma unroll
      for (int o = CL == 1 ? 8 : 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      v[k] = x;
    }
    ++sets;
    return true;
  }
  static __device__ __forceinline__ void st_async(uint32_t addr, float v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                 ::"r"(addr), "r"(__float_as_uint(v)), "r"(bar) : "memory");
  }
};

struct NormParams {
  const float* B; const float* R; const float* gate; const float* wpost; const float* wpre;
  float* Rout; float* Y; float* rstd_post; float* rstd_pre;
  // gradients
  const float* dRout; const float* dY;
  float* dR; float* dB; float* dgate;
  float* part_pre; float* part_post; float* part_gate;   // [units][M], [units][M], [units][M]
  int N, M, width, gate_rows, vecs;                      // vecs: 16-byte vectors of a row per block of the cluster
  float res_scale, scale, eps;
  // row assignment of the gradient kernel: unit u takes chunk u % chunks of gate groups
  // [u / chunks * groups_per_unit, ...), chunk_rows rows of each (chunks > 1 only with groups_per_unit == 1)
  int chunks, chunk_rows, groups_per_unit, groups;
  int gate_direct;                                       // a unit holds whole groups: deltaGate is written directly
  int units, stages, stage_bytes, slab_bytes;            // ring of the persistent kernels: rows, bytes per row / per array
  int* status;
};

// R' of one vector: res_scale R + scale gate (B rb w_post)
__device__ __forceinline__ float4 new_residual(const NormParams& p, float4 b, float4 r, float rb, float4 wpost, float4 gate) {
  float4 x = scaled(b, rb, wpost);
  x.x *= gate.x; x.y *= gate.y; x.z *= gate.z; x.w *= gate.w;
  return make_float4(fmaf(p.scale, x.x, p.res_scale * r.x), fmaf(p.scale, x.y, p.res_scale * r.y),
                     fmaf(p.scale, x.z, p.res_scale * r.z), fmaf(p.scale, x.w, p.res_scale * r.w));
}

// ------------------------------------------------------------------ forward, few rows: a row per block
// One row in flight per block, so the latency of a row counts: one vector per thread up to 4096 columns.
template <int V>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[2][32];
  BlockSum sum{slots};
  const int row = blockIdx.x;
  const long long base = static_cast<long long>(row) * p.M;
  const int vecs = p.M / 4;
  float4 b[V], r[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    b[i] = v < vecs ? clip4(ldg_row(p.B + base + v * 4), v * 4, p.width) : zero4();
    r[i] = v < vecs ? clip4(ldg_row(p.R + base + v * 4), v * 4, p.width) : zero4();
  }
  const float inv_width = 1.0f / static_cast<float>(p.width);
  float rb = 1.0f;
  if (p.wpost != nullptr) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += square_sum(b[i]);
    rb = inv_root(fmaf(sum(s), inv_width, p.eps));
    if (p.rstd_post != nullptr && threadIdx.x == 0) p.rstd_post[row] = rb;
  }
  const float* gate = p.gate == nullptr ? nullptr : p.gate + static_cast<long long>(row / p.gate_rows) * p.M;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < vecs) {
      r[i] = new_residual(p, b[i], r[i], rb, p.wpost ? load_weight(p.wpost, v, p.width) : ones4(),
                          gate ? load_weight(gate, v, p.width) : ones4());
      *reinterpret_cast<float4*>(p.Rout + base + v * 4) = r[i];
      s += square_sum(r[i]);
    }
  }
  const float rr = inv_root(fmaf(sum(s), inv_width, p.eps));
  if (p.rstd_pre != nullptr && threadIdx.x == 0) p.rstd_pre[row] = rr;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < vecs) *reinterpret_cast<float4*>(p.Y + base + v * 4) = scaled(r[i], rr, load_weight(p.wpre, v, p.width));
  }
  if (!all_finite(rb + rr + p.scale + p.res_scale)) {
    clear_padding(p.Rout + base, 0, vecs, p.width);
    clear_padding(p.Y + base, 0, vecs, p.width);
  }
}

// ------------------------------------------------------------------ ring of rows in shared memory
constexpr int MAX_STAGES = 6;
constexpr int ROLE_NORM_ROW = 8, ROLE_NORM_SUM = 9;     // what was waited for in vain, in the status word

struct RingBars {
  uint64_t full[MAX_STAGES], team[2];
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const float* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// Sets up the barriers and clears the K-value slots; every thread of the cluster returns when they can be used.
template <int CL, int K>
__device__ __forceinline__ void ring_setup(RingBars* bars, volatile int* abort_flag, float (*slots)[K][64]) {
  for (int i = threadIdx.x; i < 2 * K * 64; i += blockDim.x) (&slots[0][0][0])[i] = 0.0f;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < MAX_STAGES; ++i) mbar_init(smem_u32(&bars->full[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&bars->team[i]), CL == 1 ? blockDim.x >> 5 : 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (CL > 1) cluster_sync();
}

// The ring of A arrays per row.  refill() is for thread 0 alone, after a team sum that every warp took part in after it
// had read the place that is filled again.
template <int A>
struct Ring {
  const NormParams& p;
  RingBars* bars;
  volatile int* abort_flag;
  uint32_t base, part_bytes;
  long long part_offset;
  uint32_t read_at = 0, read_ph = 0, fill_at = 0, filled = 0, taken = 0;

  __device__ __forceinline__ void refill(const float* const (&src)[A], int row) {
    const uint32_t bar = smem_u32(&bars->full[fill_at]);
    uint32_t bytes = 0;
#pragma unroll
    for (int k = 0; k < A; ++k) bytes += src[k] != nullptr ? part_bytes : 0u;
    mbar_arrive_expect_tx(bar, bytes);
    const long long at = static_cast<long long>(row) * p.M + part_offset;
#pragma unroll
    for (int k = 0; k < A; ++k)
      if (src[k] != nullptr) bulk_load(base + fill_at * p.stage_bytes + k * p.slab_bytes, src[k] + at, part_bytes, bar);
    if (++fill_at == static_cast<uint32_t>(p.stages)) fill_at = 0;
    ++filled;
  }
  // the next row's place, once its data is there; 0 when the wait ran out
  __device__ __forceinline__ uint32_t take() {
    if (!mbar_wait(smem_u32(&bars->full[read_at]), read_ph, abort_flag)) return 0u;
    const uint32_t at = base + read_at * p.stage_bytes;
    if (++read_at == static_cast<uint32_t>(p.stages)) { read_at = 0; read_ph ^= 1u; }
    ++taken;
    return at;
  }
  // after a give-up: copies in flight land before the block may leave (thread 0, bounded)
  __device__ __forceinline__ void land() {
    for (; taken < filled; ++taken) {
      const long long t0 = clock64();
      while (!mbar_try_wait(smem_u32(&bars->full[taken % p.stages]), (taken / p.stages) & 1u) && clock64() - t0 < 20000000LL) {
      }
    }
  }
};

__device__ __forceinline__ void give_up(const NormParams& p, volatile int* abort_flag, int role, int row) {
  *abort_flag = 1;
  if ((threadIdx.x & 31) == 0) atomicCAS(p.status, 0, (role << 24) | (row & 0xFFFF));
}

// ------------------------------------------------------------------ forward, many rows
// The block (cluster) takes rows unit, unit + units, ...
template <int CL>
__global__ void __launch_bounds__(RING_THREADS, 2) norm_forward_ring_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) RingBars bars;
  __shared__ float slots[2][1][64];
  __shared__ volatile int abort_flag;
  ring_setup<CL, 1>(&bars, &abort_flag, slots);
  const int rank = CL > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / CL;
  const int vec0 = rank * p.vecs, vecs = min(p.vecs, p.M / 4 - vec0);     // this block's part of the row
  const int T = blockDim.x;
  const bool post = p.wpost != nullptr;
  const float* const src[2] = {p.B, p.R};
  Ring<2> ring{p, &bars, &abort_flag, smem_u32(ring_smem), static_cast<uint32_t>(vecs * 16), vec0 * 4};
  int fill_row = unit;
  if (threadIdx.x == 0)
    for (int i = 0; i < p.stages && fill_row < p.N; ++i, fill_row += p.units) ring.refill(src, fill_row);
  TeamSum<1, CL> sum{slots, bars.team, &abort_flag};
  const float inv_width = 1.0f / static_cast<float>(p.width);
  float4 wpre[VPT], wpost[VPT], gate[VPT];
  int gate_row = -1;                // which row of the gate is held
  bool gate_new = false;            // and has just been asked for: its columns >= width are not cleared yet
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * T + threadIdx.x;
    wpre[i] = v < vecs ? load_weight(p.wpre, vec0 + v, p.width) : zero4();
    wpost[i] = post && v < vecs ? load_weight(p.wpost, vec0 + v, p.width) : ones4();
    gate[i] = ones4();
  }
  // A row's gate is asked for behind the last stores of the row before it and cleared where it is used: with gates for 512
  // of 8192 x 2052 rows (nearly every row of a unit has another) 52 us, waiting for it at the row's start 64 us.
  auto ask_gate = [&](int for_row) {
    if (p.gate == nullptr || for_row >= p.N || for_row / p.gate_rows == gate_row) return;
    gate_row = for_row / p.gate_rows;
    gate_new = true;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      if (v < vecs) gate[i] = __ldg(reinterpret_cast<const float4*>(p.gate + static_cast<long long>(gate_row) * p.M) + vec0 + v);
    }
  };
  int row = unit, lost = 0;
  ask_gate(row);
  for (; row < p.N; row += p.units) {
    const uint32_t at = ring.take();
    if (at == 0u) { lost = ROLE_NORM_ROW; break; }
    float4 b[VPT], r[VPT];
    float t[1] = {0.0f}, rb = 1.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      b[i] = v < vecs ? clip4(lds4(at + v * 16), (vec0 + v) * 4, p.width) : zero4();
      r[i] = v < vecs ? clip4(lds4(at + p.slab_bytes + v * 16), (vec0 + v) * 4, p.width) : zero4();
      t[0] += square_sum(b[i]);
    }
    if (post) {
      if (!sum(t)) { lost = ROLE_NORM_SUM; break; }
      rb = inv_root(fmaf(t[0], inv_width, p.eps));
      if (threadIdx.x == 0) {
        if (fill_row < p.N) { ring.refill(src, fill_row); fill_row += p.units; }
        if (p.rstd_post != nullptr && rank == 0) p.rstd_post[row] = rb;
      }
    }
    const long long base = static_cast<long long>(row) * p.M + vec0 * 4;
    t[0] = 0.0f;
    if (gate_new) {
      gate_new = false;
#pragma unroll
      for (int i = 0; i < VPT; ++i) gate[i] = clip4(gate[i], (vec0 + i * T + threadIdx.x) * 4, p.width);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      r[i] = new_residual(p, b[i], r[i], rb, wpost[i], gate[i]);
      if (v < vecs) *reinterpret_cast<float4*>(p.Rout + base + v * 4) = r[i];
      t[0] += square_sum(r[i]);
    }
    if (!sum(t)) { lost = ROLE_NORM_SUM; break; }
    const float rr = inv_root(fmaf(t[0], inv_width, p.eps));
    if (threadIdx.x == 0) {
      if (!post && fill_row < p.N) { ring.refill(src, fill_row); fill_row += p.units; }
      if (p.rstd_pre != nullptr && rank == 0) p.rstd_pre[row] = rr;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      if (v < vecs) *reinterpret_cast<float4*>(p.Y + base + v * 4) = scaled(r[i], rr, wpre[i]);
    }
    if (!all_finite(rb + rr + p.scale + p.res_scale)) {
      clear_padding(p.Rout + base, vec0, vecs, p.width);
      clear_padding(p.Y + base, vec0, vecs, p.width);
    }
    ask_gate(row + p.units);
  }
  if (lost) {
    give_up(p, &abort_flag, lost, row);
    if (threadIdx.x == 0) ring.land();
    if (CL > 1) linger();
  }
  __syncthreads();
  if (CL > 1) cluster_sync();
}

// ------------------------------------------------------------------ gradients
// The rows of a unit in order: whole gate groups, or a chunk of one.
struct UnitRows {
  const NormParams& p;
  int g, g_last, row, row_end, unit;
  __device__ __forceinline__ UnitRows(const NormParams& q, int u) : p(q), unit(u) {
    g = u / p.chunks * p.groups_per_unit - 1;
    g_last = min(g + 1 + p.groups_per_unit, p.groups) - 1;
    row = row_end = 0;
  }
  // next row, or -1; g is then its group
  __device__ __forceinline__ int next() {
    while (row >= row_end) {
      if (g >= g_last) return -1;
      ++g;
      const long long first = static_cast<long long>(g) * p.gate_rows + static_cast<long long>(unit % p.chunks) * p.chunk_rows;
      const long long end = min(min(static_cast<long long>(g + 1) * p.gate_rows, first + p.chunk_rows), static_cast<long long>(p.N));
      row = static_cast<int>(min(first, end));
      row_end = static_cast<int>(end);
    }
    return row++;
  }
};

// The ring holds deltaY, R', B and deltaR' of a row.  What the outputs need of a row beside its sums are three values per
// element, a = deltaR' + q / rms(R'), r^ / rms(R') and b^: they stay in registers over the reduction.
template <int CL, bool POST, bool GATE>
__global__ void __launch_bounds__(DELTA_BOUND) norm_delta_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) RingBars bars;
  __shared__ float slots[2][3][64];
  __shared__ volatile int abort_flag;
  ring_setup<CL, 3>(&bars, &abort_flag, slots);
  const int rank = CL > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / CL;
  const int vec0 = rank * p.vecs, vecs = min(p.vecs, p.M / 4 - vec0);
  const int T = blockDim.x;
  const float* const src[4] = {p.dY, p.Rout, p.B, p.dRout};
  Ring<4> ring{p, &bars, &abort_flag, smem_u32(ring_smem), static_cast<uint32_t>(vecs * 16), vec0 * 4};
  UnitRows fill_rows(p, unit);
  if (threadIdx.x == 0)
    for (int i = 0, row; i < p.stages && (row = fill_rows.next()) >= 0; ++i) ring.refill(src, row);
  // the column sums' blocks may take their places as this grid's blocks leave (they wait for its end before they read)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  TeamSum<3, CL> sum{slots, bars.team, &abort_flag};
  const float inv_width = 1.0f / static_cast<float>(p.width);
  const bool has_dr = p.dRout != nullptr;
  float4 wpre[VPT], wpost[VPT], gate[VPT], dwpre[VPT], dwpost[VPT], dgate[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * T + threadIdx.x;
    wpre[i] = v < vecs ? load_weight(p.wpre, vec0 + v, p.width) : zero4();
    wpost[i] = POST && v < vecs ? load_weight(p.wpost, vec0 + v, p.width) : ones4();
    gate[i] = ones4();
    dwpre[i] = dwpost[i] = dgate[i] = zero4();
  }
  UnitRows rows(p, unit);
  int row = rows.next(), group = -1, lost = 0;
  bool gate_new = false;                       // asked for as in the forward kernel
  auto ask_gate = [&](int g) {
    if (!GATE || g == group) return;
    group = g;
    gate_new = true;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      if (v < vecs) gate[i] = __ldg(reinterpret_cast<const float4*>(p.gate + static_cast<long long>(g) * p.M) + vec0 + v);
    }
  };
  if (row >= 0) ask_gate(rows.g);
  float rb = POST && row >= 0 ? __ldg(p.rstd_post + row) : 1.0f, rr = row >= 0 ? __ldg(p.rstd_pre + row) : 0.0f;
  while (row >= 0) {
    const int next_row = rows.next();
    float next_rb = 1.0f, next_rr = 0.0f;      // a row ahead
    if (next_row >= 0) {
      if (POST) next_rb = __ldg(p.rstd_post + next_row);
      next_rr = __ldg(p.rstd_pre + next_row);
    }
    const uint32_t at0 = ring.take();
    if (at0 == 0u) { lost = ROLE_NORM_ROW; break; }
    if (GATE && gate_new) {
      gate_new = false;
#pragma unroll
      for (int i = 0; i < VPT; ++i) gate[i] = clip4(gate[i], (vec0 + i * T + threadIdx.x) * 4, p.width);
    }
    float4 a[VPT], c[VPT], b[VPT];
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      a[i] = c[i] = b[i] = zero4();
      if (v < vecs) {
        const uint32_t at = at0 + v * 16;
        const int col = (vec0 + v) * 4;
        const float4 dy = clip4(lds4(at), col, p.width);
        const float4 ro = clip4(lds4(at + p.slab_bytes), col, p.width);
        b[i] = clip4(lds4(at + 2 * p.slab_bytes), col, p.width);
        if (has_dr) a[i] = clip4(lds4(at + 3 * p.slab_bytes), col, p.width);
        auto one = [&](float dyv, float rv, float& av, float& cv, float& bv, float g, float w, float wo, float& dw) {
          const float r = rv * rr, q = dyv * w;
          if (POST) bv *= rb;
          cv = r * rr;
          av = fmaf(rr, q, av);
          dw = fmaf(dyv, r, dw);
          s[0] = fmaf(q, r, s[0]);
          if (POST) {
            const float e = p.scale * g * wo * bv;
            s[1] = fmaf(e, av, s[1]);
            s[2] = fmaf(e, cv, s[2]);
          }
        };
        one(dy.x, ro.x, a[i].x, c[i].x, b[i].x, gate[i].x, wpre[i].x, wpost[i].x, dwpre[i].x);
        one(dy.y, ro.y, a[i].y, c[i].y, b[i].y, gate[i].y, wpre[i].y, wpost[i].y, dwpre[i].y);
        one(dy.z, ro.z, a[i].z, c[i].z, b[i].z, gate[i].z, wpre[i].z, wpost[i].z, dwpre[i].z);
        one(dy.w, ro.w, a[i].w, c[i].w, b[i].w, gate[i].w, wpre[i].w, wpost[i].w, dwpre[i].w);
      }
    }
    if (!sum(s)) { lost = ROLE_NORM_SUM; break; }
    if (threadIdx.x == 0) {
      const int more = fill_rows.next();
      if (more >= 0) ring.refill(src, more);
    }
    const float c1 = s[0] * inv_width, c2 = fmaf(-c1, s[2], s[1]) * inv_width;
    const long long base = static_cast<long long>(row) * p.M + vec0 * 4;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      if (v < vecs) {
        float4 odr, odb;
        auto one = [&](float av, float cv, float bv, float g, float wo, float& o_dr, float& o_db, float& dpost, float& dgt) {
          const float dT = fmaf(-cv, c1, av);
          const float dP = p.scale * g * dT;
          o_dr = p.res_scale * dT;
          o_db = POST ? rb * fmaf(-bv, c2, dP * wo) : dP;
          if (POST) dpost = fmaf(dP, bv, dpost);
          if (GATE) dgt = fmaf(p.scale * bv * wo, dT, dgt);
        };
        one(a[i].x, c[i].x, b[i].x, gate[i].x, wpost[i].x, odr.x, odb.x, dwpost[i].x, dgate[i].x);
        one(a[i].y, c[i].y, b[i].y, gate[i].y, wpost[i].y, odr.y, odb.y, dwpost[i].y, dgate[i].y);
        one(a[i].z, c[i].z, b[i].z, gate[i].z, wpost[i].z, odr.z, odb.z, dwpost[i].z, dgate[i].z);
        one(a[i].w, c[i].w, b[i].w, gate[i].w, wpost[i].w, odr.w, odb.w, dwpost[i].w, dgate[i].w);
        *reinterpret_cast<float4*>(p.dR + base + v * 4) = odr;     // padding columns: the column sums' kernel clears them
        *reinterpret_cast<float4*>(p.dB + base + v * 4) = odb;
      }
    }
    if (GATE && p.gate_direct && (next_row < 0 || rows.g != group)) {     // the group's rows are done
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        if (v < vecs)
          *reinterpret_cast<float4*>(p.dgate + static_cast<long long>(group) * p.M + (vec0 + v) * 4) =
              clip4(dgate[i], (vec0 + v) * 4, p.width);
        dgate[i] = zero4();
      }
    }
    if (next_row >= 0) ask_gate(rows.g);
    row = next_row; rb = next_rb; rr = next_rr;
  }
  if (lost) {
    give_up(p, &abort_flag, lost, row);
    if (threadIdx.x == 0) ring.land();
    if (CL > 1) linger();
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = i * T + threadIdx.x;
    if (v < vecs) {
      const long long at = static_cast<long long>(unit) * p.M + (vec0 + v) * 4;
      *reinterpret_cast<float4*>(p.part_pre + at) = dwpre[i];
      if (POST) *reinterpret_cast<float4*>(p.part_post + at) = dwpost[i];
      if (GATE && !p.gate_direct) *reinterpret_cast<float4*>(p.part_gate + at) = dgate[i];
    }
  }
  __syncthreads();
  if (CL > 1) cluster_sync();
}

// ------------------------------------------------------------------ column sums of the units' partial rows
struct ColSumParams {
  const float* in[3];
  float* out[3];
  int rows[3];      // partial rows per output row
  int M, width, N, groups;
  float* rows_out[2];    // deltaR, deltaB: columns >= width are set to zeros here, because a row whose sums are not finite
                         // leaves NaN there (looking at it in the rows' kernel cost wide rows 5 to 10 % of its time)
};
// Block: 8 vectors of columns x 32 slices of the rows; blockIdx.y = output row, blockIdx.z = which sum.
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ ColSumParams p) {
  __shared__ float4 part[32][8];
  const int z = blockIdx.z;
  const float* in = p.in[z];
  const bool sums = in != nullptr && static_cast<int>(blockIdx.y) < (z < 2 ? 1 : p.groups);
  if (!sums && z > 0) return;
  const int c = threadIdx.x & 7, slice = threadIdx.x >> 3;
  const int v = blockIdx.x * 8 + c;
  const int rows = p.rows[z];
  float4 s = zero4();
  asm volatile("griddepcontrol.wait;" ::: "memory");      // the partial rows are complete
  if (z == 0 && p.width < p.M) {
    const int warps = gridDim.x * gridDim.y * 8, warp = (blockIdx.y * gridDim.x + blockIdx.x) * 8 + (threadIdx.x >> 5);
    for (int row = warp; row < p.N; row += warps)
      for (int col = p.width + (threadIdx.x & 31); col < p.M; col += 32) {
        const long long at = static_cast<long long>(row) * p.M + col;
        p.rows_out[0][at] = 0.0f;
        p.rows_out[1][at] = 0.0f;
      }
  }
  if (!sums) return;
  if (v < p.M / 4) {
    const float4* src = reinterpret_cast<const float4*>(in) + static_cast<long long>(blockIdx.y) * rows * (p.M / 4) + v;
#pragma unroll 4
    for (int r = slice; r < rows; r += 32) {
      const float4 x = src[static_cast<long long>(r) * (p.M / 4)];
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
  }
  part[slice][c] = s;
  __syncthreads();
  if (threadIdx.x < 8 && v < p.M / 4) {
    for (int k = 1; k < 32; ++k) {
      const float4 x = part[k][c];
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    reinterpret_cast<float4*>(p.out[z])[static_cast<long long>(blockIdx.y) * (p.M / 4) + v] = clip4(s, v * 4, p.width);
  }
}

// ------------------------------------------------------------------ host
// How a row of M floats is laid on a persistent kernel: blocks per row, vectors per block, working threads, and a ring of
// rows of `arrays` parts that leaves room for the blocks an SM takes.
constexpr int FORWARD_REGS = 64, DELTA_REGS = 96;      // what the kernels are compiled to at their launch bounds
constexpr int FORWARD_SMEM = 640, DELTA_SMEM = 1664;   // their shared memory beside the ring
// What an SM has: registers for a warp's 32 threads in each of its four parts, and shared memory, of which every block costs
// 1 KB more than it asks for.
constexpr int SM_PART_REGS = 16384, SM_SMEM = 228 * 1024, BLOCK_SMEM = 1024, SM_BLOCKS = 32;
constexpr int MOST_RING = 220 * 1024;                  // dynamic shared memory of a block
// A plan takes 220 KB and 2 KB per block beside the rings: what is left of the 228 KB is the L1 cache's (8192 x 1136, both
// calls: 80 us; filled to the brim 89).
constexpr int PLAN_SMEM = 220 * 1024, PLAN_BLOCK = 2048;
struct Shape { int cl, vecs, threads, stages, stage_bytes, slab_bytes, per_sm; };

Shape ring_shape(int M, int arrays, int regs, int smem) {
  Shape s{};
  const int all = M / 4;
  s.cl = all <= 1024 ? 1 : (all <= 2048 ? 2 : 4);
  s.vecs = (all + s.cl - 1) / s.cl;
  s.threads = ((s.vecs + VPT - 1) / VPT + 31) / 32 * 32;
  s.slab_bytes = s.vecs * 16;
  s.stage_bytes = (s.slab_bytes * arrays + 127) / 128 * 128;
  // Blocks per SM: by shared memory and by the registers per thread.  Three rows in a ring, but two in a cluster's, whose
  // exchange of sums a second block covers better than a third row (gradients of 8192 x 5000: 161 us, with three 213;
  // single blocks of 256 columns: 52 us with three, 63 with two).
  // No more than are resident at a time: a block left over would start when one of the others has done all its rows (gradients
  // of 8192 x 620, 6 blocks to an SM, with the forward: 55 us, planned with 7: 62).
  auto least = [](int a, int b) { return a < b ? a : b; };
  const int ring = (s.cl == 1 ? 3 : 2) * s.stage_bytes, fixed = smem + BLOCK_SMEM;
  const int by_smem = least(PLAN_SMEM / (ring + PLAN_BLOCK), SM_SMEM / (ring + fixed));
  const int by_regs = 4 * (SM_PART_REGS / (regs * 32)) / (s.threads / 32);
  s.per_sm = least(least(by_smem, by_regs), SM_BLOCKS);
  if (s.per_sm < 1) s.per_sm = 1;
  s.stages = least(PLAN_SMEM / s.per_sm - PLAN_BLOCK, SM_SMEM / s.per_sm - fixed) / s.stage_bytes;
  s.stages = least(s.stages, MAX_STAGES);
  return s;
}

// Clusters of the given size that run at the same time, each block with a whole SM (asked once per device).
template <int CL>
int cluster_count() {
  static std::atomic<int> cache[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return device_sm_count() / CL;
  int n = cache[dev & 63].load(std::memory_order_acquire);
  if (n > 0) return n;
  cudaLaunchConfig_t q = {};
  q.gridDim = dim3(static_cast<unsigned>(device_sm_count() / CL * CL), 1, 1);
  q.blockDim = dim3(RING_THREADS, 1, 1);
  q.dynamicSmemBytes = 210 * 1024;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  q.attrs = attr;
  q.numAttrs = 1;
  if (cudaFuncSetAttribute(norm_delta_kernel<CL, true, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_RING) !=
          cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, norm_delta_kernel<CL, true, true>, &q) != cudaSuccess || n < 1) {
    cudaGetLastError();      // no device, or none that could run it: the launch will say so
    return device_sm_count() / CL > 0 ? device_sm_count() / CL : 1;
  }
  cache[dev & 63].store(n, std::memory_order_release);
  return n;
}

// Blocks (clusters) that fill the device once.
int ring_units(const Shape& s) {
  if (s.cl == 1) return device_sm_count() * s.per_sm;
  return (s.cl == 2 ? cluster_count<2>() : cluster_count<4>()) * s.per_sm;
}

template <void (*kernel)(NormParams)>
cudaError_t launch_ring(const Shape& s, NormParams p, cudaStream_t st) {
  static std::atomic<int> ready[64];      // per device and kernel: the shared-memory opt-in has been made
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_RING);
    if (e != cudaSuccess) return e;
    ready[dev & 63].store(1, std::memory_order_release);
  }
  p.status = status_word_ptr(&e);
  if (!p.status) return e;
  p.vecs = s.vecs; p.stages = s.stages; p.stage_bytes = s.stage_bytes; p.slab_bytes = s.slab_bytes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.units) * s.cl, 1, 1);
  cfg.blockDim = dim3(s.threads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(s.stages) * s.stage_bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(s.cl);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.cl > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int CL>
cudaError_t launch_delta(bool post, bool gate, const Shape& s, const NormParams& p, cudaStream_t st) {
  if (post && gate) return launch_ring<norm_delta_kernel<CL, true, true>>(s, p, st);
  if (post) return launch_ring<norm_delta_kernel<CL, true, false>>(s, p, st);
  if (gate) return launch_ring<norm_delta_kernel<CL, false, true>>(s, p, st);
  return launch_ring<norm_delta_kernel<CL, false, false>>(s, p, st);
}

// How the gradient kernel's units share the rows.
struct RowPlan { int units, chunks, chunk_rows, groups_per_unit, groups, gate_rows; bool direct; };

RowPlan plan_rows(int N, int gate_rows, int want) {
  RowPlan r{};
  r.gate_rows = gate_rows > 0 && gate_rows < N ? gate_rows : N;
  r.groups = (N + r.gate_rows - 1) / r.gate_rows;
  if (want < 1) want = 1;
  if (r.groups >= want) {
    r.groups_per_unit = (r.groups + want - 1) / want;
    r.units = (r.groups + r.groups_per_unit - 1) / r.groups_per_unit;
    r.chunks = 1; r.chunk_rows = r.gate_rows; r.direct = true;
  } else {
    int chunks = want / r.groups;
    if (chunks > r.gate_rows) chunks = r.gate_rows;
    r.chunk_rows = (r.gate_rows + chunks - 1) / chunks;
    r.chunks = (r.gate_rows + r.chunk_rows - 1) / r.chunk_rows;
    r.groups_per_unit = 1;
    r.units = r.groups * r.chunks;
    r.direct = r.chunks == 1;
  }
  return r;
}

long long work_floats_of(const RowPlan& r, int M) { return static_cast<long long>(r.units) * M * 3; }

int check_rows(int N, int M, int width, int gate_rows) {
  if (N <= 0 || M <= 0 || width <= 0 || width > M || M > MAX_WIDTH || gate_rows < 0) return CU32_E_DIM;
  if (static_cast<long long>(N) * 4 >= (1LL << 31)) return CU32_E_DIM;
  if (M & 3) return CU32_E_ALIGN;
  return CU32_OK;
}

template <class... P>
bool any_null(const P*... p) { return (... || (p == nullptr)); }
template <class... P>
bool all_aligned16(const P*... p) { return (... && aligned16(p)); }

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

int cu32_normResidual(int64_t stream, const float* B, const float* R, const float* gate, int gate_rows, const float* wpost,
                      const float* wpre, float* Rout, float* Y, float* rstd_post, float* rstd_pre, int N, int M, int width,
                      float res_scale, float scale, float eps) {
  if (any_null(B, R, wpre, Rout, Y)) return CU32_E_NULL;
  if (int rc = check_rows(N, M, width, gate_rows)) return rc;
  if (gate && gate_rows == 0) return CU32_E_DIM;
  if (!(eps >= 0.0f)) return CU32_E_ARG;
  if (!all_aligned16(B, R, gate, wpost, wpre, Rout, Y)) return CU32_E_ALIGN;
  NormParams p{};
  p.B = B; p.R = R; p.gate = gate; p.wpost = wpost; p.wpre = wpre; p.Rout = Rout; p.Y = Y;
  p.rstd_post = rstd_post; p.rstd_pre = rstd_pre;
  p.N = N; p.M = M; p.width = width; p.gate_rows = gate_rows > 0 ? gate_rows : 1;
  p.res_scale = res_scale; p.scale = scale; p.eps = eps;
  const cudaStream_t st = as_stream(stream);
  // Up to two rows per SM a block of its own for each row is the faster form: no ring to fill, one vector per thread.
  if (N <= 2 * device_sm_count()) {
    const int vecs = M / 4;
    const int threads = vecs >= 1024 ? 1024 : (vecs + 31) / 32 * 32;
    if (vecs <= 1024) norm_forward_kernel<1><<<N, threads, 0, st>>>(p);
    else norm_forward_kernel<4><<<N, threads, 0, st>>>(p);
    return static_cast<int>(cudaPeekAtLastError());
  }
  const Shape s = ring_shape(M, 2, FORWARD_REGS, FORWARD_SMEM);
  p.units = ring_units(s);
  if (p.units > N) p.units = N;
  if (s.cl == 1) return static_cast<int>(launch_ring<norm_forward_ring_kernel<1>>(s, p, st));
  if (s.cl == 2) return static_cast<int>(launch_ring<norm_forward_ring_kernel<2>>(s, p, st));
  return static_cast<int>(launch_ring<norm_forward_ring_kernel<4>>(s, p, st));
}

long long cu32_normResidual_work(int N, int M, int gate_rows) {
  if (check_rows(N, M, M, gate_rows)) return 0;
  return work_floats_of(plan_rows(N, gate_rows, ring_units(ring_shape(M, 4, DELTA_REGS, DELTA_SMEM))), M);
}

int cu32_normResidual_delta(int64_t stream, const float* dRout, const float* dY, const float* B, const float* Rout,
                            const float* gate, int gate_rows, const float* wpost, const float* wpre, const float* rstd_post,
                            const float* rstd_pre, float* dR, float* dB, float* dgate, float* dwpost, float* dwpre,
                            float* work, long long work_floats, int N, int M, int width, float res_scale, float scale) {
  if (any_null(dY, B, Rout, wpre, rstd_pre, dR, dB, dwpre, work)) return CU32_E_NULL;
  if ((wpost && any_null(rstd_post, dwpost)) || (gate && !dgate)) return CU32_E_NULL;
  if (int rc = check_rows(N, M, width, gate_rows)) return rc;
  if (gate && gate_rows == 0) return CU32_E_DIM;
  if (!all_aligned16(dRout, dY, B, Rout, gate, wpost, wpre, dR, dB, dgate, dwpost, dwpre, work)) return CU32_E_ALIGN;
  const Shape s = ring_shape(M, 4, DELTA_REGS, DELTA_SMEM);
  int want = ring_units(s);
  const long long room = work_floats / (3LL * M);
  if (room < 1) return CU32_E_SCRATCH;
  if (want > room) want = static_cast<int>(room);
  const RowPlan r = plan_rows(N, gate ? gate_rows : 0, want);
  if (work_floats_of(r, M) > work_floats) return CU32_E_SCRATCH;
  NormParams p{};
  p.B = B; p.gate = gate; p.wpost = wpost; p.wpre = wpre; p.Rout = const_cast<float*>(Rout);
  p.rstd_post = const_cast<float*>(rstd_post); p.rstd_pre = const_cast<float*>(rstd_pre);
  p.dRout = dRout; p.dY = dY; p.dR = dR; p.dB = dB; p.dgate = dgate;
  const long long rows = static_cast<long long>(r.units) * M;
  p.part_pre = work; p.part_post = work + rows; p.part_gate = work + 2 * rows;
  p.N = N; p.M = M; p.width = width; p.units = r.units;
  p.res_scale = res_scale; p.scale = scale;
  p.chunks = r.chunks; p.chunk_rows = r.chunk_rows; p.groups_per_unit = r.groups_per_unit; p.groups = r.groups;
  p.gate_rows = r.gate_rows; p.gate_direct = r.direct ? 1 : 0;
  const cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (s.cl == 1) e = launch_delta<1>(wpost != nullptr, gate != nullptr, s, p, st);
  else if (s.cl == 2) e = launch_delta<2>(wpost != nullptr, gate != nullptr, s, p, st);
  else e = launch_delta<4>(wpost != nullptr, gate != nullptr, s, p, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  ColSumParams c{};
  c.M = M; c.width = width; c.N = N;
  c.rows_out[0] = dR; c.rows_out[1] = dB;
  c.in[0] = p.part_pre; c.out[0] = dwpre; c.rows[0] = r.units;
  if (wpost) { c.in[1] = p.part_post; c.out[1] = dwpost; c.rows[1] = r.units; }
  const bool gate_sum = gate && !r.direct;
  if (gate_sum) { c.in[2] = p.part_gate; c.out[2] = dgate; c.rows[2] = r.chunks; }
  c.groups = r.groups;
  const int across = (M / 4 + 7) / 8;
  int down = gate_sum ? r.groups : 1;
  if (width < M) {      // a warp clears some 16 rows
    int clear = (N / 128 + across - 1) / across;
    const int most = 8 * device_sm_count() / across;
    if (clear > most) clear = most;
    if (down < clear) down = clear;
  }
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(down), gate_sum ? 3u : 2u);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, column_sum_kernel, c));
}

}  // extern "C"
