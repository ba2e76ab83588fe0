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
// than 4096 columns, each block a part of the row) with a producer warp that brings the next rows into a ring in shared
// memory by bulk copies while the others compute, so that loads are in flight all the time whatever the row's
// reductions wait for.  The column sums are kept in registers over all rows of a block, written once per block and added
// in a fixed order by a second, small kernel (no atomics: results do not vary from run to run).
#include <atomic>

#include "cu32_host.h"

namespace dragon {
namespace {

using namespace ptx;

constexpr int MAX_WIDTH = 16384;     // floats per row: a cluster of four blocks of 1024 vectors
constexpr int VPT = 2;               // 16-byte vectors per thread of the persistent kernels

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

__device__ __forceinline__ float4 ones4() { return make_float4(1.f, 1.f, 1.f, 1.f); }
__device__ __forceinline__ float square_sum(float4 v) { return v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w; }
__device__ __forceinline__ float4 scaled(float4 v, float f, float4 w) {
  return make_float4(v.x * f * w.x, v.y * f * w.y, v.z * f * w.z, v.w * f * w.w);
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

// Sums of K values over the working warps of the blocks of a cluster, in two steps: post() publishes this warp's sums and
// returns at once, wait() delivers the totals of the oldest posted set.  Two sets may be open (the slots alternate): a
// warp posts set i + 2 only after its wait for set i + 1, which every warp posted after it had read set i.
template <int K, int CL>
struct TeamSum {
  float (*slots)[K][64];      // [2][K][64]: by set parity, value, warp of the cluster (at most 16 per block)
  uint64_t* bars;             // [2], one arrival per warp of the cluster
  volatile int* abort_flag;
  int warps;                  // working warps per block
  uint32_t posted = 0, taken = 0;

  __device__ __forceinline__ void post(float (&v)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int par = posted & 1;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (CL == 1) {
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) slots[par][k][warp] = v[k];
        mbar_arrive(smem_u32(&bars[par]));
      }
    } else if (lane < CL) {     // lane r delivers to block r
      const int at = static_cast<int>(cluster_ctarank()) * warps + warp;
#pragma unroll
      for (int k = 0; k < K; ++k) st_cluster(mapa(smem_u32(&slots[par][k][at]), lane), v[k]);
      mbar_arrive_cluster_release(mapa(smem_u32(&bars[par]), lane));
    }
    ++posted;
  }
  __device__ __forceinline__ bool wait(float (&v)[K]) {
    const int lane = threadIdx.x & 31;
    const int par = taken & 1;
    if (!mbar_wait<(CL > 1)>(smem_u32(&bars[par]), (taken >> 1) & 1u, abort_flag)) return false;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float x = lane < warps * CL ? slots[par][k][lane] : 0.0f;
      if (CL > 2 && lane + 32 < warps * CL) x += slots[par][k][lane + 32];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      v[k] = x;
    }
    ++taken;
    return true;
  }
  static __device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
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
__device__ __forceinline__ float4 new_residual(const NormParams& p, float4 b, float4 r, float rb, float4 wpost,
                                               const float* gate, int v) {
  float4 x = scaled(b, rb, wpost);
  if (gate != nullptr) {
    const float4 g = load_weight(gate, v, p.width);
    x.x *= g.x; x.y *= g.y; x.z *= g.z; x.w *= g.w;
  }
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
    rb = 1.0f / sqrtf(fmaf(sum(s), inv_width, p.eps));
    if (p.rstd_post != nullptr && threadIdx.x == 0) p.rstd_post[row] = rb;
  }
  const float* gate = p.gate == nullptr ? nullptr : p.gate + static_cast<long long>(row / p.gate_rows) * p.M;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < vecs) {
      r[i] = new_residual(p, b[i], r[i], rb, p.wpost ? load_weight(p.wpost, v, p.width) : ones4(), gate, v);
      *reinterpret_cast<float4*>(p.Rout + base + v * 4) = r[i];
      s += square_sum(r[i]);
    }
  }
  const float rr = 1.0f / sqrtf(fmaf(sum(s), inv_width, p.eps));
  if (p.rstd_pre != nullptr && threadIdx.x == 0) p.rstd_pre[row] = rr;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = i * blockDim.x + threadIdx.x;
    if (v < vecs) *reinterpret_cast<float4*>(p.Y + base + v * 4) = scaled(r[i], rr, load_weight(p.wpre, v, p.width));
  }
}

// ------------------------------------------------------------------ ring of rows in shared memory
constexpr int MAX_STAGES = 4;
constexpr int ROLE_NORM_PRODUCER = 8, ROLE_NORM_ROW = 9;     // who gave up, in the status word

struct RingBars {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], team[2];
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
__device__ __forceinline__ void give_up(const NormParams& p, volatile int* abort_flag, int role, uint32_t it) {
  *abort_flag = 1;
  atomicCAS(p.status, 0, (role << 24) | static_cast<int>(it & 0xFFFF));
}

// Sets up the barriers; every thread of the cluster returns when they can be used.
template <int CL>
__device__ __forceinline__ void ring_setup(RingBars* bars, volatile int* abort_flag, int warps) {
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(smem_u32(&bars->full[i]), 1);
      mbar_init(smem_u32(&bars->empty[i]), warps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&bars->team[i]), warps * CL);
    fence_mbar_init();
  }
  __syncthreads();
  if (CL > 1) cluster_sync();
}

// One thread: copies `arrays` row parts per row into the ring, rows in the order that next() gives them (-1: the end).
template <class Next>
__device__ __forceinline__ void produce(const NormParams& p, RingBars* bars, volatile int* abort_flag, uint32_t ring,
                                        const float* const (&src)[4], uint32_t part_bytes, long long part_offset, Next next) {
  uint32_t it = 0, s = 0, ph = 0;
  for (long long row; (row = next()) >= 0; ++it) {
    if (!mbar_wait(smem_u32(&bars->empty[s]), ph ^ 1u, abort_flag)) {
      give_up(p, abort_flag, ROLE_NORM_PRODUCER, it);
      break;
    }
    const uint32_t bar = smem_u32(&bars->full[s]);
    uint32_t bytes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) bytes += src[k] != nullptr ? part_bytes : 0u;
    mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (src[k] != nullptr)
        bulk_load(ring + s * p.stage_bytes + k * p.slab_bytes, src[k] + row * p.M + part_offset, part_bytes, bar);
    if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1u; }
  }
  if (*abort_flag) {     // copies in flight land before the block may leave
    const uint32_t n = it < static_cast<uint32_t>(p.stages) ? it : static_cast<uint32_t>(p.stages);
    for (uint32_t k = 0; k < n; ++k) {
      const uint32_t i = it - n + k;
      const long long t0 = clock64();
      while (!mbar_try_wait(smem_u32(&bars->full[i % p.stages]), (i / p.stages) & 1u) && clock64() - t0 < 20000000LL) {
      }
    }
  }
}

// ------------------------------------------------------------------ forward, many rows
// Block: the working warps, then one producer warp.  The block (cluster) takes rows unit, unit + units, ...
template <int CL>
__global__ void __launch_bounds__(544) norm_forward_ring_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) RingBars bars;
  __shared__ float slots[2][1][64];
  __shared__ volatile int abort_flag;
  const int warps = (blockDim.x >> 5) - 1;
  ring_setup<CL>(&bars, &abort_flag, warps);
  const int rank = CL > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / CL;
  const int vec0 = rank * p.vecs, vecs = min(p.vecs, p.M / 4 - vec0);     // this block's part of the row
  const uint32_t ring = smem_u32(ring_smem);
  if ((threadIdx.x >> 5) == warps) {
    if ((threadIdx.x & 31) == 0) {
      const float* const src[4] = {p.B, p.R, nullptr, nullptr};
      long long row = unit - p.units;
      produce(p, &bars, &abort_flag, ring, src, vecs * 16, vec0 * 4, [&]() -> long long {
        row += p.units;
        return row < p.N ? row : -1;
      });
    }
  } else {
    TeamSum<1, CL> team{slots, bars.team, &abort_flag, warps};
    const int T = warps * 32;
    const float inv_width = 1.0f / static_cast<float>(p.width);
    float4 wpre[VPT], wpost[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      wpre[i] = v < vecs ? load_weight(p.wpre, vec0 + v, p.width) : zero4();
      wpost[i] = v < vecs && p.wpost ? load_weight(p.wpost, vec0 + v, p.width) : ones4();
    }
    uint32_t s = 0, ph = 0;
    for (int row = unit; row < p.N; row += p.units) {
      if (!mbar_wait(smem_u32(&bars.full[s]), ph, &abort_flag)) {
        give_up(p, &abort_flag, ROLE_NORM_ROW, row);
        break;
      }
      float4 b[VPT], r[VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        const uint32_t at = ring + s * p.stage_bytes + v * 16;
        b[i] = v < vecs ? clip4(lds4(at), (vec0 + v) * 4, p.width) : zero4();
        r[i] = v < vecs ? clip4(lds4(at + p.slab_bytes), (vec0 + v) * 4, p.width) : zero4();
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&bars.empty[s]));     // the row is in registers
      if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1u; }
      float rb = 1.0f, t[1];
      if (p.wpost != nullptr) {
        t[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) t[0] += square_sum(b[i]);
        team.post(t);
        if (!team.wait(t)) { give_up(p, &abort_flag, ROLE_NORM_ROW, row); break; }
        rb = 1.0f / sqrtf(fmaf(t[0], inv_width, p.eps));
        if (p.rstd_post != nullptr && threadIdx.x == 0 && rank == 0) p.rstd_post[row] = rb;
      }
      const long long base = static_cast<long long>(row) * p.M + vec0 * 4;
      const float* gate = p.gate == nullptr ? nullptr : p.gate + static_cast<long long>(row / p.gate_rows) * p.M;
      t[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        if (v < vecs) {
          r[i] = new_residual(p, b[i], r[i], rb, wpost[i], gate, vec0 + v);
          *reinterpret_cast<float4*>(p.Rout + base + v * 4) = r[i];
          t[0] += square_sum(r[i]);
        }
      }
      team.post(t);
      if (!team.wait(t)) { give_up(p, &abort_flag, ROLE_NORM_ROW, row); break; }
      const float rr = 1.0f / sqrtf(fmaf(t[0], inv_width, p.eps));
      if (p.rstd_pre != nullptr && threadIdx.x == 0 && rank == 0) p.rstd_pre[row] = rr;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        if (v < vecs) *reinterpret_cast<float4*>(p.Y + base + v * 4) = scaled(r[i], rr, wpre[i]);
      }
    }
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

// Block: the working warps, then one producer warp; the ring holds deltaY, R', B and deltaR' of a row.  The sums of
// row i + 1 are formed and posted before the outputs of row i are, so nobody stands at a barrier for a row's reduction.
template <int CL, bool POST, bool GATE>
__global__ void __launch_bounds__(544) norm_delta_kernel(const __grid_constant__ NormParams p) {
  extern __shared__ __align__(128) uint8_t ring_smem[];
  __shared__ __align__(8) RingBars bars;
  __shared__ float slots[2][3][64];
  __shared__ volatile int abort_flag;
  const int warps = (blockDim.x >> 5) - 1;
  ring_setup<CL>(&bars, &abort_flag, warps);
  const int rank = CL > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / CL;
  const int vec0 = rank * p.vecs, vecs = min(p.vecs, p.M / 4 - vec0);
  const uint32_t ring = smem_u32(ring_smem);
  if ((threadIdx.x >> 5) == warps) {
    if ((threadIdx.x & 31) == 0) {
      const float* const src[4] = {p.dY, p.Rout, p.B, p.dRout};
      UnitRows rows(p, unit);
      produce(p, &bars, &abort_flag, ring, src, vecs * 16, vec0 * 4, [&]() -> long long { return rows.next(); });
    }
  } else {
    TeamSum<3, CL> team{slots, bars.team, &abort_flag, warps};
    const int T = warps * 32;
    const float inv_width = 1.0f / static_cast<float>(p.width);
    const bool has_dr = p.dRout != nullptr;
    float4 wpre[VPT], wpost[VPT], dwpre[VPT], dwpost[VPT], dgate[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = i * T + threadIdx.x;
      wpre[i] = v < vecs ? load_weight(p.wpre, vec0 + v, p.width) : zero4();
      wpost[i] = POST && v < vecs ? load_weight(p.wpost, vec0 + v, p.width) : ones4();
      dwpre[i] = dwpost[i] = dgate[i] = zero4();
    }
    struct Row { int row, g; float rb, rr; };
    UnitRows rows(p, unit);
    auto fetch = [&]() -> Row {       // the next row's index and its two factors, which are needed a row later
      Row x;
      x.row = rows.next();
      x.g = rows.g;
      x.rb = 1.0f; x.rr = 0.0f;
      if (x.row >= 0) {
        if (POST) x.rb = __ldg(p.rstd_post + x.row);
        x.rr = __ldg(p.rstd_pre + x.row);
      }
      return x;
    };
    auto gate_at = [&](int g, int v) { return load_weight(p.gate + static_cast<long long>(g) * p.M, vec0 + v, p.width); };
    // q r^, e (deltaR' + q / rms), e r^ / rms summed over the row; also deltaW_pre
    auto sums_of = [&](const Row& x, uint32_t stage, float (&s)[3]) {
      s[0] = s[1] = s[2] = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        if (v < vecs) {
          const uint32_t at = ring + stage * p.stage_bytes + v * 16;
          const int col = (vec0 + v) * 4;
          const float4 dy = clip4(lds4(at), col, p.width);
          const float4 ro = clip4(lds4(at + p.slab_bytes), col, p.width);
          float4 b = zero4(), dr = zero4(), gt = ones4();
          if (POST) {
            b = clip4(lds4(at + 2 * p.slab_bytes), col, p.width);
            if (has_dr) dr = clip4(lds4(at + 3 * p.slab_bytes), col, p.width);
            if (GATE) gt = gate_at(x.g, v);
          }
          auto one = [&](float dyv, float rv, float bv, float drv, float g, float w, float wo, float& dw) {
            const float r = rv * x.rr, q = dyv * w;
            dw = fmaf(dyv, r, dw);
            s[0] = fmaf(q, r, s[0]);
            if (POST) {
              const float e = p.scale * g * wo * (bv * x.rb);
              s[1] = fmaf(e, fmaf(x.rr, q, drv), s[1]);
              s[2] = fmaf(e * x.rr, r, s[2]);
            }
          };
          one(dy.x, ro.x, b.x, dr.x, gt.x, wpre[i].x, wpost[i].x, dwpre[i].x);
          one(dy.y, ro.y, b.y, dr.y, gt.y, wpre[i].y, wpost[i].y, dwpre[i].y);
          one(dy.z, ro.z, b.z, dr.z, gt.z, wpre[i].z, wpost[i].z, dwpre[i].z);
          one(dy.w, ro.w, b.w, dr.w, gt.w, wpre[i].w, wpost[i].w, dwpre[i].w);
        }
      }
    };
    // deltaR, deltaB of the row; deltaW_post and deltaGate
    auto outputs_of = [&](const Row& x, uint32_t stage, float c1, float c2) {
      const long long base = static_cast<long long>(x.row) * p.M + vec0 * 4;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = i * T + threadIdx.x;
        if (v < vecs) {
          const uint32_t at = ring + stage * p.stage_bytes + v * 16;
          const int col = (vec0 + v) * 4;
          const float4 dy = clip4(lds4(at), col, p.width);
          const float4 ro = clip4(lds4(at + p.slab_bytes), col, p.width);
          const float4 b = POST || GATE ? clip4(lds4(at + 2 * p.slab_bytes), col, p.width) : zero4();
          const float4 dr = has_dr ? clip4(lds4(at + 3 * p.slab_bytes), col, p.width) : zero4();
          const float4 gt = GATE ? gate_at(x.g, v) : ones4();
          float4 odr, odb;
          auto one = [&](float dyv, float rv, float bv, float drv, float g, float w, float wo, float& o_dr, float& o_db,
                         float& dpost, float& dgt) {
            const float bh = POST ? bv * x.rb : bv;
            const float dT = fmaf(x.rr, fmaf(-(rv * x.rr), c1, dyv * w), drv);
            const float dP = p.scale * g * dT;
            o_dr = p.res_scale * dT;
            if (POST) {
              o_db = x.rb * fmaf(-bh, c2, dP * wo);
              dpost = fmaf(dP, bh, dpost);
            } else {
              o_db = dP;
            }
            if (GATE) dgt = fmaf(p.scale * bh * wo, dT, dgt);
          };
          one(dy.x, ro.x, b.x, dr.x, gt.x, wpre[i].x, wpost[i].x, odr.x, odb.x, dwpost[i].x, dgate[i].x);
          one(dy.y, ro.y, b.y, dr.y, gt.y, wpre[i].y, wpost[i].y, odr.y, odb.y, dwpost[i].y, dgate[i].y);
          one(dy.z, ro.z, b.z, dr.z, gt.z, wpre[i].z, wpost[i].z, odr.z, odb.z, dwpost[i].z, dgate[i].z);
          one(dy.w, ro.w, b.w, dr.w, gt.w, wpre[i].w, wpost[i].w, odr.w, odb.w, dwpost[i].w, dgate[i].w);
          *reinterpret_cast<float4*>(p.dR + base + v * 4) = odr;     // padding columns: every operand was cleared
          *reinterpret_cast<float4*>(p.dB + base + v * 4) = odb;
        }
      }
    };
    uint32_t s = 0, ph = 0;           // ring position of the row whose sums come next
    auto advance = [&]() { if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1u; } };
    Row cur = fetch(), nxt = fetch();
    float t[3], c[3];
    uint32_t stage = 0;
    bool alive = cur.row >= 0;
    if (alive) {
      alive = mbar_wait(smem_u32(&bars.full[s]), ph, &abort_flag);
      if (alive) {
        sums_of(cur, s, t);
        team.post(t);
        stage = s;
        advance();
        alive = team.wait(c);
      }
    }
    while (alive && cur.row >= 0) {
      const uint32_t next_stage = s;
      const Row after = nxt.row >= 0 ? fetch() : nxt;
      if (nxt.row >= 0) {
        alive = mbar_wait(smem_u32(&bars.full[s]), ph, &abort_flag);
        if (!alive) break;
        sums_of(nxt, s, t);
        team.post(t);
        advance();
      }
      const float c1 = c[0] * inv_width;
      outputs_of(cur, stage, c1, fmaf(-c1, c[2], c[1]) * inv_width);
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(&bars.empty[stage]));
      if (GATE && p.gate_direct && (nxt.row < 0 || nxt.g != cur.g)) {     // the group's rows are done
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int v = i * T + threadIdx.x;
          if (v < vecs) *reinterpret_cast<float4*>(p.dgate + static_cast<long long>(cur.g) * p.M + (vec0 + v) * 4) = dgate[i];
          dgate[i] = zero4();
        }
      }
      if (nxt.row >= 0) alive = team.wait(c);
      cur = nxt;
      nxt = after;
      stage = next_stage;
    }
    if (!alive && cur.row >= 0 && (threadIdx.x & 31) == 0) give_up(p, &abort_flag, ROLE_NORM_ROW, cur.row);
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
  }
  __syncthreads();
  if (CL > 1) cluster_sync();
}

// ------------------------------------------------------------------ column sums of the units' partial rows
struct ColSumParams {
  const float* in[3];
  float* out[3];
  int rows[3];      // partial rows per output row
  int M;
};
// Block: 8 vectors of columns x 32 slices of the rows; blockIdx.y = output row, blockIdx.z = which sum.
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ ColSumParams p) {
  __shared__ float4 part[32][8];
  const int z = blockIdx.z;
  const float* in = p.in[z];
  if (in == nullptr || (z < 2 && blockIdx.y > 0)) return;
  const int c = threadIdx.x & 7, slice = threadIdx.x >> 3;
  const int v = blockIdx.x * 8 + c;
  const int rows = p.rows[z];
  float4 s = zero4();
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
    reinterpret_cast<float4*>(p.out[z])[static_cast<long long>(blockIdx.y) * (p.M / 4) + v] = s;
  }
}

// ------------------------------------------------------------------ host
// How a row of M floats is laid on a persistent kernel: blocks per row, vectors per block, working threads, and a ring of
// rows of `arrays` parts that leaves room for the blocks an SM takes.
struct Shape { int cl, vecs, threads, stages, stage_bytes, slab_bytes, per_sm; };

Shape ring_shape(int M, int arrays) {
  Shape s{};
  const int all = M / 4;
  s.cl = all <= 1024 ? 1 : (all <= 2048 ? 2 : 4);
  s.vecs = (all + s.cl - 1) / s.cl;
  s.threads = ((s.vecs + VPT - 1) / VPT + 31) / 32 * 32;
  s.slab_bytes = s.vecs * 16;
  s.stage_bytes = (s.slab_bytes * arrays + 127) / 128 * 128;
  // blocks per SM: by shared memory at three rows each, by registers (at most 112 per thread: 544 threads fit once)
  const int by_smem = 220 * 1024 / (3 * s.stage_bytes + 2048), by_regs = 585 / (s.threads + 32);
  s.per_sm = by_smem < by_regs ? by_smem : by_regs;
  if (s.per_sm < 1) s.per_sm = 1;
  s.stages = (220 * 1024 / s.per_sm - 2048) / s.stage_bytes;
  if (s.stages > MAX_STAGES) s.stages = MAX_STAGES;
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
  q.blockDim = dim3(544, 1, 1);
  q.dynamicSmemBytes = 210 * 1024;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  q.attrs = attr;
  q.numAttrs = 1;
  if (cudaFuncSetAttribute(norm_delta_kernel<CL, true, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) !=
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
  return s.cl == 2 ? cluster_count<2>() : cluster_count<4>();
}

template <void (*kernel)(NormParams)>
cudaError_t launch_ring(const Shape& s, NormParams p, cudaStream_t st) {
  static std::atomic<int> ready[64];      // per device and kernel: the shared-memory opt-in has been made
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
    if (e != cudaSuccess) return e;
    ready[dev & 63].store(1, std::memory_order_release);
  }
  p.status = status_word_ptr(&e);
  if (!p.status) return e;
  p.vecs = s.vecs; p.stages = s.stages; p.stage_bytes = s.stage_bytes; p.slab_bytes = s.slab_bytes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.units) * s.cl, 1, 1);
  cfg.blockDim = dim3(s.threads + 32, 1, 1);
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
  const Shape s = ring_shape(M, 2);
  p.units = ring_units(s);
  if (p.units > N) p.units = N;
  if (s.cl == 1) return static_cast<int>(launch_ring<norm_forward_ring_kernel<1>>(s, p, st));
  if (s.cl == 2) return static_cast<int>(launch_ring<norm_forward_ring_kernel<2>>(s, p, st));
  return static_cast<int>(launch_ring<norm_forward_ring_kernel<4>>(s, p, st));
}

long long cu32_normResidual_work(int N, int M, int gate_rows) {
  if (check_rows(N, M, M, gate_rows)) return 0;
  return work_floats_of(plan_rows(N, gate_rows, ring_units(ring_shape(M, 4))), M);
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
  const Shape s = ring_shape(M, 4);
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
  c.M = M;
  c.in[0] = p.part_pre; c.out[0] = dwpre; c.rows[0] = r.units;
  if (wpost) { c.in[1] = p.part_post; c.out[1] = dwpost; c.rows[1] = r.units; }
  const bool gate_sum = gate && !r.direct;
  if (gate_sum) { c.in[2] = p.part_gate; c.out[2] = dgate; c.rows[2] = r.chunks; }
  const dim3 grid(static_cast<unsigned>((M / 4 + 7) / 8), gate_sum ? static_cast<unsigned>(r.groups) : 1u, gate_sum ? 3u : 2u);
  column_sum_kernel<<<grid, 256, 0, st>>>(c);
  return static_cast<int>(cudaPeekAtLastError());
}

}  // extern "C"
