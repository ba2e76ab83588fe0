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
// Bound by memory: forward 4 floats per element (B, R in; R', Y out), gradients 6 (four in, two out).  A row lives in the
// registers of one thread block (a cluster of two or four for the widest), so nothing is read twice; the column sums
// are kept in registers over all rows of the block, written once per block and added in a fixed order by a second,
// small kernel (no atomics: results do not vary from run to run).
#include <cooperative_groups.h>
#include <atomic>

#include "cu32_host.h"

namespace dragon {
namespace {

namespace cg = cooperative_groups;

constexpr int MAX_WIDTH = 16384;     // floats per row: four blocks of 1024 vectors

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

// Sums of K values over the threads of the block (CL > 1: over the blocks of the cluster), the same in every thread.
// One barrier per call: the slots alternate, so a slot is written again only after everybody has passed the barrier of
// the call in between.  Warps of all blocks: at most 32.
template <int K, int CL>
struct TeamSum {
  float (*slots)[K][32];     // [2][K][32]
  int parity = 0;
  __device__ __forceinline__ void operator()(float (&v)[K]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (CL == 1 && warps == 1) return;
    const int rank = CL > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
    if (lane < K) {
      float mine = v[0];
#pragma unroll
      for (int k = 1; k < K; ++k) mine = lane == k ? v[k] : mine;
      float* slot = &slots[parity][lane][rank * warps + warp];
      if (CL == 1) *slot = mine;
      else
        for (int r = 0; r < CL; ++r) *cg::this_cluster().map_shared_rank(slot, r) = mine;
    }
    if (CL == 1) __syncthreads();
    else cg::this_cluster().sync();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = lane < warps * CL ? slots[parity][k][lane] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      v[k] = s;
    }
    parity ^= 1;
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
};

// ------------------------------------------------------------------ forward: one row per block (or cluster)
template <int VPT, int CL>
__global__ void __launch_bounds__(1024) norm_forward_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[2][1][32];
  TeamSum<1, CL> sum{slots};
  const int rank = CL > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
  if (CL > 1) cg::this_cluster().sync();     // the other blocks' slots exist from here on
  const int row = blockIdx.x / CL;
  const long long base = static_cast<long long>(row) * p.M;
  const int last_vec = min((rank + 1) * p.vecs, p.M / 4);
  float4 b[VPT], r[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = rank * p.vecs + i * blockDim.x + threadIdx.x;
    const bool ok = v < last_vec;
    b[i] = ok ? clip4(ldg_row(p.B + base + v * 4), v * 4, p.width) : zero4();
    r[i] = ok ? clip4(ldg_row(p.R + base + v * 4), v * 4, p.width) : zero4();
  }
  const float inv_width = 1.0f / static_cast<float>(p.width);
  float rb = 1.0f;
  if (p.wpost != nullptr) {
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[0] += b[i].x * b[i].x + b[i].y * b[i].y + b[i].z * b[i].z + b[i].w * b[i].w;
    sum(s);
    rb = 1.0f / sqrtf(fmaf(s[0], inv_width, p.eps));
    if (p.rstd_post != nullptr && threadIdx.x == 0 && rank == 0) p.rstd_post[row] = rb;
  }
  const float* gate = p.gate == nullptr ? nullptr : p.gate + static_cast<long long>(row / p.gate_rows) * p.M;
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = rank * p.vecs + i * blockDim.x + threadIdx.x;
    if (v < last_vec) {
      float4 x = b[i];
      if (p.wpost != nullptr) {
        const float4 w = clip4(__ldg(reinterpret_cast<const float4*>(p.wpost) + v), v * 4, p.width);
        x.x = x.x * rb * w.x; x.y = x.y * rb * w.y; x.z = x.z * rb * w.z; x.w = x.w * rb * w.w;
      }
      if (gate != nullptr) {
        const float4 g = clip4(__ldg(reinterpret_cast<const float4*>(gate) + v), v * 4, p.width);
        x.x *= g.x; x.y *= g.y; x.z *= g.z; x.w *= g.w;
      }
      r[i].x = fmaf(p.scale, x.x, p.res_scale * r[i].x); r[i].y = fmaf(p.scale, x.y, p.res_scale * r[i].y);
      r[i].z = fmaf(p.scale, x.z, p.res_scale * r[i].z); r[i].w = fmaf(p.scale, x.w, p.res_scale * r[i].w);
      *reinterpret_cast<float4*>(p.Rout + base + v * 4) = r[i];
      s[0] += r[i].x * r[i].x + r[i].y * r[i].y + r[i].z * r[i].z + r[i].w * r[i].w;
    }
  }
  sum(s);
  const float rr = 1.0f / sqrtf(fmaf(s[0], inv_width, p.eps));
  if (p.rstd_pre != nullptr && threadIdx.x == 0 && rank == 0) p.rstd_pre[row] = rr;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = rank * p.vecs + i * blockDim.x + threadIdx.x;
    if (v < last_vec) {
      const float4 w = clip4(__ldg(reinterpret_cast<const float4*>(p.wpre) + v), v * 4, p.width);
      *reinterpret_cast<float4*>(p.Y + base + v * 4) =
          make_float4(r[i].x * rr * w.x, r[i].y * rr * w.y, r[i].z * rr * w.z, r[i].w * rr * w.w);
    }
  }
}

// ------------------------------------------------------------------ gradients: a unit (block or cluster) per run of rows
template <int VPT, int CL, bool POST, bool GATE>
__global__ void __launch_bounds__(256) norm_delta_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[2][3][32];
  TeamSum<3, CL> sum{slots};
  const int rank = CL > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
  if (CL > 1) cg::this_cluster().sync();
  const int unit = blockIdx.x / CL;
  const int last_vec = min((rank + 1) * p.vecs, p.M / 4);
  const float inv_width = 1.0f / static_cast<float>(p.width);
  const int v0 = rank * p.vecs + threadIdx.x;
  float4 dwpre[VPT], dwpost[POST ? VPT : 1], dgate[GATE ? VPT : 1];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    dwpre[i] = zero4();
    if (POST) dwpost[i] = zero4();
    if (GATE) dgate[i] = zero4();
  }
  const int g_first = unit / p.chunks * p.groups_per_unit;
  const int g_last = min(g_first + p.groups_per_unit, p.groups);
  for (int g = g_first; g < g_last; ++g) {
    const long long group0 = static_cast<long long>(g) * p.gate_rows;
    const int row_first = static_cast<int>(min(group0 + static_cast<long long>(unit % p.chunks) * p.chunk_rows, static_cast<long long>(p.N)));
    const int row_last = static_cast<int>(min(min(group0 + p.gate_rows, static_cast<long long>(row_first) + p.chunk_rows), static_cast<long long>(p.N)));
    const float* gate = GATE ? p.gate + static_cast<long long>(g) * p.M : nullptr;
    for (int row = row_first; row < row_last; ++row) {
      const long long base = static_cast<long long>(row) * p.M;
      const float rb = POST ? p.rstd_post[row] : 1.0f, rr = p.rstd_pre[row];
      float4 dy[VPT], dr[VPT], rh[VPT], bh[VPT];
      float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * blockDim.x;
        const bool ok = v < last_vec;
        const long long at = base + v * 4;
        dy[i] = ok ? clip4(ldg_row(p.dY + at), v * 4, p.width) : zero4();
        rh[i] = ok ? clip4(ldg_row(p.Rout + at), v * 4, p.width) : zero4();
        dr[i] = ok && p.dRout != nullptr ? clip4(ldg_row(p.dRout + at), v * 4, p.width) : zero4();
        bh[i] = ok ? clip4(ldg_row(p.B + at), v * 4, p.width) : zero4();
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * blockDim.x;
        if (v < last_vec) {
          const float4 wp = clip4(__ldg(reinterpret_cast<const float4*>(p.wpre) + v), v * 4, p.width);
          float4 e = make_float4(p.scale, p.scale, p.scale, p.scale);
          if (GATE) {
            const float4 gt = clip4(__ldg(reinterpret_cast<const float4*>(gate) + v), v * 4, p.width);
            e.x *= gt.x; e.y *= gt.y; e.z *= gt.z; e.w *= gt.w;
          }
          float4 wq = make_float4(1.f, 1.f, 1.f, 1.f);
          if (POST) wq = clip4(__ldg(reinterpret_cast<const float4*>(p.wpost) + v), v * 4, p.width);
          auto one = [&](float dyv, float drv, float& r, float& b, float w, float gs, float wo, float& dw) {
            r *= rr;
            if (POST) b *= rb;
            const float q = dyv * w;
            dw = fmaf(dyv, r, dw);
            s[0] = fmaf(q, r, s[0]);
            if (POST) {
              const float ev = gs * wo * b;
              s[1] = fmaf(ev, fmaf(rr, q, drv), s[1]);
              s[2] = fmaf(ev * rr, r, s[2]);
            }
          };
          one(dy[i].x, dr[i].x, rh[i].x, bh[i].x, wp.x, e.x, wq.x, dwpre[i].x);
          one(dy[i].y, dr[i].y, rh[i].y, bh[i].y, wp.y, e.y, wq.y, dwpre[i].y);
          one(dy[i].z, dr[i].z, rh[i].z, bh[i].z, wp.z, e.z, wq.z, dwpre[i].z);
          one(dy[i].w, dr[i].w, rh[i].w, bh[i].w, wp.w, e.w, wq.w, dwpre[i].w);
        }
      }
      sum(s);
      const float c1 = s[0] * inv_width;
      const float c2 = fmaf(-c1, s[2], s[1]) * inv_width;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * blockDim.x;
        if (v < last_vec) {
          const float4 wp = clip4(__ldg(reinterpret_cast<const float4*>(p.wpre) + v), v * 4, p.width);
          float4 gt = make_float4(1.f, 1.f, 1.f, 1.f);
          if (GATE) gt = clip4(__ldg(reinterpret_cast<const float4*>(gate) + v), v * 4, p.width);
          float4 wq = make_float4(1.f, 1.f, 1.f, 1.f);
          if (POST) wq = clip4(__ldg(reinterpret_cast<const float4*>(p.wpost) + v), v * 4, p.width);
          float4 odr, odb;
          auto one = [&](float dyv, float drv, float r, float b, float w, float gv, float wo, float& o_dr, float& o_db,
                         float* dpost, float* dgt) {
            const float dT = fmaf(rr, fmaf(-r, c1, dyv * w), drv);
            o_dr = p.res_scale * dT;
            const float dP = p.scale * gv * dT;
            if (POST) {
              o_db = rb * fmaf(-b, c2, dP * wo);
              *dpost = fmaf(dP, b, *dpost);
            } else {
              o_db = dP;
            }
            if (GATE) *dgt = fmaf(p.scale * (POST ? b * wo : b), dT, *dgt);
          };
          constexpr int Z = 0;
          const int ip = POST ? i : Z, ig = GATE ? i : Z;
          one(dy[i].x, dr[i].x, rh[i].x, bh[i].x, wp.x, gt.x, wq.x, odr.x, odb.x, &dwpost[ip].x, &dgate[ig].x);
          one(dy[i].y, dr[i].y, rh[i].y, bh[i].y, wp.y, gt.y, wq.y, odr.y, odb.y, &dwpost[ip].y, &dgate[ig].y);
          one(dy[i].z, dr[i].z, rh[i].z, bh[i].z, wp.z, gt.z, wq.z, odr.z, odb.z, &dwpost[ip].z, &dgate[ig].z);
          one(dy[i].w, dr[i].w, rh[i].w, bh[i].w, wp.w, gt.w, wq.w, odr.w, odb.w, &dwpost[ip].w, &dgate[ig].w);
          // (padding columns: every operand was cleared, so both come out 0; without w_post B's were too)
          if (p.dR != nullptr) *reinterpret_cast<float4*>(p.dR + base + v * 4) = odr;
          if (p.dB != nullptr) *reinterpret_cast<float4*>(p.dB + base + v * 4) = odb;
        }
      }
    }
    if (GATE && p.gate_direct) {     // the group's rows are done
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * blockDim.x;
        if (v < last_vec) *reinterpret_cast<float4*>(p.dgate + static_cast<long long>(g) * p.M + v * 4) = dgate[i];
        dgate[i] = zero4();
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = v0 + i * blockDim.x;
    if (v < last_vec) {
      const long long at = static_cast<long long>(unit) * p.M + v * 4;
      *reinterpret_cast<float4*>(p.part_pre + at) = dwpre[i];
      if (POST) *reinterpret_cast<float4*>(p.part_post + at) = dwpost[i];
      if (GATE && !p.gate_direct) *reinterpret_cast<float4*>(p.part_gate + at) = dgate[i];
    }
  }
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
// Threads per block, vectors per thread and blocks per row for rows of M floats.
struct Shape { int threads, vpt, cl, vecs; };

int round_warps(int threads) { return (threads + 31) / 32 * 32; }

// forward: up to 4 vectors per thread, 1024 threads
Shape forward_shape(int M, int N) {
  const int vecs = M / 4;
  Shape s{32, 1, 1, vecs};
  // few rows: the latency of a row counts, so one vector per thread; many rows: four, for the loads in flight
  const int vpt = N <= 2 * device_sm_count() ? 1 : 4;
  s.vpt = vpt;
  s.threads = round_warps((vecs + vpt - 1) / vpt);
  if (s.threads > 1024) { s.threads = 1024; s.vpt = 4; }
  return s;
}

Shape delta_shape(int M) {
  const int vecs = M / 4;
  Shape s{32, 4, 1, vecs};
  s.cl = vecs <= 1024 ? 1 : (vecs <= 2048 ? 2 : 4);
  s.vecs = (vecs + s.cl - 1) / s.cl;
  s.threads = round_warps((s.vecs + s.vpt - 1) / s.vpt);
  return s;
}

template <class K>
cudaError_t launch(K kernel, int blocks, int threads, int cl, const NormParams& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks) * cl, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cl);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cl > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int CL>
cudaError_t launch_delta(bool post, bool gate, int units, int threads, const NormParams& p, cudaStream_t st) {
  if (post && gate) return launch(norm_delta_kernel<4, CL, true, true>, units, threads, CL, p, st);
  if (post) return launch(norm_delta_kernel<4, CL, true, false>, units, threads, CL, p, st);
  if (gate) return launch(norm_delta_kernel<4, CL, false, true>, units, threads, CL, p, st);
  return launch(norm_delta_kernel<4, CL, false, false>, units, threads, CL, p, st);
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

// Units that fill the device: registers allow about 512 threads per SM.
int wanted_units(const Shape& s) {
  int per_sm = 512 / (s.threads * s.cl);
  if (per_sm < 1) per_sm = 1;
  return s.threads * s.cl > 512 ? device_sm_count() * 512 / (s.threads * s.cl) : device_sm_count() * per_sm;
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
  const Shape s = forward_shape(M, N);
  p.vecs = s.vecs;
  const cudaStream_t st = as_stream(stream);
  return static_cast<int>(s.vpt == 1 ? launch(norm_forward_kernel<1, 1>, N, s.threads, 1, p, st)
                                     : launch(norm_forward_kernel<4, 1>, N, s.threads, 1, p, st));
}

long long cu32_normResidual_work(int N, int M, int gate_rows) {
  if (check_rows(N, M, M, gate_rows)) return 0;
  return work_floats_of(plan_rows(N, gate_rows, wanted_units(delta_shape(M))), M);
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
  const Shape s = delta_shape(M);
  int want = wanted_units(s);
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
  p.N = N; p.M = M; p.width = width; p.vecs = s.vecs;
  p.res_scale = res_scale; p.scale = scale;
  p.chunks = r.chunks; p.chunk_rows = r.chunk_rows; p.groups_per_unit = r.groups_per_unit; p.groups = r.groups;
  p.gate_rows = r.gate_rows; p.gate_direct = r.direct ? 1 : 0;
  const cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (s.cl == 1) e = launch_delta<1>(wpost != nullptr, gate != nullptr, r.units, s.threads, p, st);
  else if (s.cl == 2) e = launch_delta<2>(wpost != nullptr, gate != nullptr, r.units, s.threads, p, st);
  else e = launch_delta<4>(wpost != nullptr, gate != nullptr, r.units, s.threads, p, st);
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
