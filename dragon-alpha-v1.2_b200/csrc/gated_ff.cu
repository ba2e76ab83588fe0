// Gated feed-forward block:  H = act(X Wg) * (X Wu),  Y = H Wd,  and its gradients.
//
//   X [N, D], Wg, Wu [D, F], Wd [F, D]; G = X Wg, U = X Wu.
//   deltaH = deltaY Wd^T;  deltaG = deltaH * U * act'(G);  deltaU = deltaH * act(G)
//   deltaX = deltaG Wg^T + deltaU Wu^T;  deltaWg = X^T deltaG;  deltaWu = X^T deltaU;  deltaWd = H^T deltaY
//
// Three forms, by what bounds them:
// Up to 8 rows, forward: every weight is read once for all rows by FP32 multiply-adds, so the time is that of reading
//   3 D F floats (rows_kernel below; 4096 / 10924, 537 MB: 92 us for one row, 102 us for 8, in a long graph; a call by
//   itself 109 to 113 us for 8).  The multiply-adds fill the issue slots beyond: 16 rows would take as long as two calls.
// Up to 128 rows: the same reading bounds it, but the products run on the tensor cores with the weights as the tile's
//   rows (gemm_thin.cu; 16 rows 119 us, 128 rows 264 us, where the tiles below took 315 and 320 us with a cut second
//   product); it needs scratch, without it these calls take 490 to 500 us.  The gradients use it from one row on, with all
//   weight gradients in one launch up to 24 rows (gated_outer.cu).
// More rows: the contraction kernel (gemm_tf32.cuh) with both projections in one launch and act(G) * U formed in the
//   registers that hold the sums, and with the two products of deltaX in one accumulation.  6 N D F flop forward and
//   12 N D F backward at the FP32-accurate rate bound it.
#include <atomic>
#include <initializer_list>

#include "cu32_host.h"
#include "gated_thin.h"

namespace dragon {
namespace {

using namespace ptx;

// ------------------------------------------------------------------ few rows
struct RowsParams {
  CUtensorMap tmW[2];         // [K, M] weights, boxes of KT rows x CPW columns; the second only for the gated form
  CUtensorMap tmX;            // [N, K] operand, boxes of NR rows x KT columns
  float* out;                 // [N, M]
  float* G;                   // gated form: pre-activations, or null
  float* U;
  int N, M, act;
  int ktiles, items, clusters, stages;
  int early;                  // the grid may start before the one that writes X has ended
  int give_up;                // tests: w + 1, or ROWS_WARPS + w + 1: worker warp w of block 0 loses its first wait for a tile,
                              // or for an item's sums; 0: none
  int* status;
};

constexpr int ROWS_WARPS = 8, ROWS_WORKERS = ROWS_WARPS * 32, ROWS_THREADS = ROWS_WORKERS + 32;
constexpr int ROWS_MAX_STAGES = 12;
constexpr int ROLE_ROWS_LOAD = 10, ROLE_ROWS_TILE = 11, ROLE_ROWS_SUM = 12;

__device__ __forceinline__ float4 lds_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts_v4(uint32_t addr, float4 v) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// Pairs of floats in one 64-bit register: fma.rn.f32x2 does both products in one issue, at twice the scalar rate.
typedef unsigned long long f32x2;
__device__ __forceinline__ void lds_pairs(uint32_t addr, f32x2& a, f32x2& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr));
}
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
__device__ __forceinline__ float2 lds_v2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
// 16 bytes to a block of the cluster, counted by that block's barrier
__device__ __forceinline__ void st_async_v4(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(addr), "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)),
                 "r"(__float_as_uint(v.w)), "r"(bar) : "memory");
}
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(ROWS_WORKERS) : "memory"); }

// Shared memory of a block: [ring of tiles][sums of the warps, four rows at a time][inbox, two items]
template <int NR, int MATS, int CPW, int S>
struct RowsCfg {
  static constexpr int KT = 4096 / CPW;                                 // rows of the weights per tile: 16 KB a matrix
  static constexpr int W_BYTES = KT * CPW * 4, X_BYTES = NR * KT * 4;
  static constexpr int TILE_BYTES = MATS * W_BYTES + (X_BYTES + 127) / 128 * 128;
  static constexpr int GROUP = NR < 4 ? NR : 4;                         // rows reduced at a time
  static constexpr int RED_BYTES = ROWS_WARPS * GROUP * MATS * CPW * 4;
  static constexpr int BOX_BYTES = NR * MATS * CPW * 4;                 // an item's sums from all blocks of the cluster
  static constexpr int FIXED = RED_BYTES + 2 * BOX_BYTES + 128;
  static constexpr int STAGES_FIT = (224 * 1024 - FIXED) / TILE_BYTES;
  static constexpr int STAGES = STAGES_FIT < ROWS_MAX_STAGES ? STAGES_FIT : ROWS_MAX_STAGES;
  static constexpr int SMEM = FIXED + STAGES * TILE_BYTES;
  static_assert(STAGES >= 3, "ring");
};

// out[n, :] = X[n, :] W  (MATS = 1)  or  act(X[n, :] W0) * (X[n, :] W1)  (MATS = 2)  for N <= NR rows.
// The weights are read once for all rows: the time is theirs.  A producer warp keeps a ring of weight tiles (KT rows x CPW
// columns, with the KT columns of X that meet them) full by TMA whatever the workers do; the persistent cluster takes
// blocks of CPW columns in turn, its S blocks a slice of K each.  A worker holds 4 columns x NR rows of sums; the sums of
// lanes, warps and blocks are added in a fixed order, each block of the cluster finishing CPW / S columns.
// (Measured for 8 rows of a 4096 / 10924 block, 537 MB: 102 us in a long graph, 5.2 TB/s, and 109 us, 4.9 TB/s, for calls one
// by one; with plain loads into registers instead of the ring, one launch over all column blocks, 184 us.)
template <int NR, int MATS, int CPW, int S>
__global__ void __launch_bounds__(ROWS_THREADS, 1) rows_kernel(const __grid_constant__ RowsParams p) {
  using Cfg = RowsCfg<NR, MATS, CPW, S>;
  extern __shared__ __align__(128) uint8_t rows_smem[];
  __shared__ __align__(8) uint64_t bar_full[ROWS_MAX_STAGES], bar_empty[ROWS_MAX_STAGES], bar_box[2];
  __shared__ volatile int abort_flag, lost[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = S > 1 ? cluster_ctarank() : 0u;
  const uint32_t ring = (smem_u32(rows_smem) + 127u) & ~127u;
  const uint32_t red = ring + Cfg::STAGES * Cfg::TILE_BYTES, box = red + Cfg::RED_BYTES;
  if (threadIdx.x == 0) {
    abort_flag = lost[0] = lost[1] = 0;
    for (int i = 0; i < ROWS_MAX_STAGES; ++i) {
      mbar_init(smem_u32(&bar_full[i]), 1);
      mbar_init(smem_u32(&bar_empty[i]), ROWS_WARPS);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&bar_box[i]), 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (S > 1) cluster_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int first_item = blockIdx.x / S;
  const int t0 = static_cast<int>(rank) * p.ktiles / S, t1 = (static_cast<int>(rank) + 1) * p.ktiles / S;
  auto give_up = [&](int role, int it) {
    abort_flag = 1;
    atomicCAS(p.status, 0, (role << 24) | (it & 0xFFFF));
  };

  if (warp == ROWS_WARPS) {
    if (lane == 0) {
      // Weight tiles may be on their way before X exists: only X's loads wait for the grid that writes it.
      auto load_w = [&](uint32_t st, int item, int t) {
        const uint32_t bar = smem_u32(&bar_full[st]), dst = ring + st * Cfg::TILE_BYTES;
        mbar_arrive_expect_tx(bar, MATS * Cfg::W_BYTES + Cfg::X_BYTES);
#pragma unroll
        for (int m = 0; m < MATS; ++m) tma_load_3d(dst + m * Cfg::W_BYTES, &p.tmW[m], bar, item * CPW, t * Cfg::KT, 0, 0ull);
      };
      auto load_x = [&](uint32_t st, int t) {
        tma_load_3d(ring + st * Cfg::TILE_BYTES + MATS * Cfg::W_BYTES, &p.tmX, smem_u32(&bar_full[st]), t * Cfg::KT, 0, 0, 0ull);
      };
      uint32_t st = 0, ph = 0, it = 0;
      int early_x[ROWS_MAX_STAGES];
      int held = 0;                        // tiles whose X has not been asked for yet
      bool started = p.early == 0, alive = true;
      for (int item = first_item; alive && item < p.items; item += p.clusters) {
        for (int t = t0; t < t1; ++t, ++it) {
          if (!started && held == Cfg::STAGES) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (int i = 0; i < held; ++i) load_x(i, early_x[i]);
            started = true;
          }
          if (!mbar_wait(smem_u32(&bar_empty[st]), ph ^ 1u, &abort_flag)) {
            give_up(ROLE_ROWS_LOAD, it);
            alive = false;
            break;
          }
          load_w(st, item, t);
          if (started) load_x(st, t);
          else early_x[held++] = t;
          if (++st == Cfg::STAGES) { st = 0; ph ^= 1u; }
        }
      }
      if (!started) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int i = 0; i < held; ++i) load_x(i, early_x[i]);
      }
      if (abort_flag) {                    // copies in flight land before the block may leave
        const uint32_t n = it < static_cast<uint32_t>(Cfg::STAGES) ? it : static_cast<uint32_t>(Cfg::STAGES);
        for (uint32_t i = it - n; i < it; ++i) {
          const long long c0 = clock64();
          while (!mbar_try_wait(smem_u32(&bar_full[i % Cfg::STAGES]), (i / Cfg::STAGES) & 1u) && clock64() - c0 < 20000000LL) {
          }
        }
      }
    }
  } else {
    constexpr int LPR = CPW / 4;           // lanes per row of the tile
    constexpr int RPL = 4;                 // rows of the tile per lane
    const int k_in = (warp * (32 / LPR) + lane / LPR) * RPL, c_in = (lane % LPR) * 4;
    uint32_t st = 0, ph = 0, done = 0;
    const int loses = blockIdx.x == 0 ? p.give_up - 1 - warp : -1;
    // A wait may run out in one warp and succeed in another a moment later.  Whoever lost one says so and goes on to the next
    // barrier of the workers all the same, behind which all of them look and leave together: nobody waits at a barrier for
    // warps that have left.  There are two such barriers per item, each with a word of its own, so that a warp that is ahead
    // says nothing yet where another still has to look.
    bool alive = true;
    for (int item = first_item; alive && item < p.items; item += p.clusters, ++done) {
      f32x2 acc2[NR][MATS][2];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MATS; ++m) acc2[n][m][0] = acc2[n][m][1] = 0ull;
      // A lane's four rows of a tile go in two parts of two; the loads of a part are under way during the products of the
      // part before it, across tiles too, and a tile is given back as soon as its second part has been read.
      constexpr int JB = RPL / 2;
      struct Part { f32x2 w[JB][MATS][2]; float2 x[NR]; };
      auto load = [&](Part& q, uint32_t tile, int j0) {
#pragma unroll
        for (int j = 0; j < JB; ++j)
#pragma unroll
          for (int m = 0; m < MATS; ++m)
            lds_pairs(tile + m * Cfg::W_BYTES + ((k_in + j0 + j) * CPW + c_in) * 4, q.w[j][m][0], q.w[j][m][1]);
#pragma unroll
        for (int n = 0; n < NR; ++n) q.x[n] = lds_v2(tile + MATS * Cfg::W_BYTES + (n * Cfg::KT + k_in + j0) * 4);
      };
      auto multiply = [&](const Part& q) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int j = 0; j < JB; ++j) {
            const f32x2 x = both(j == 0 ? q.x[n].x : q.x[n].y);
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
              fma_pair(acc2[n][m][0], x, q.w[j][m][0]);
              fma_pair(acc2[n][m][1], x, q.w[j][m][1]);
            }
          }
      };
      auto arrived = [&](int t, bool loses_it) {
        if (!loses_it && mbar_wait(smem_u32(&bar_full[st]), ph, &abort_flag)) return true;
        if (lane == 0) give_up(ROLE_ROWS_TILE, t);
        return false;
      };
      Part a, b;
      alive = arrived(t0, loses == 0);
      if (alive) load(a, ring + st * Cfg::TILE_BYTES, 0);
      for (int t = t0; alive && t < t1; ++t) {
        load(b, ring + st * Cfg::TILE_BYTES, JB);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_empty[st]));
        if (++st == Cfg::STAGES) { st = 0; ph ^= 1u; }
        multiply(a);
        if (t + 1 < t1) {
          alive = arrived(t + 1, false);
          if (alive) load(a, ring + st * Cfg::TILE_BYTES, 0);
        }
        multiply(b);
      }
      if (!alive) {
        lost[0] = 1;
        workers_sync();
        break;
      }
      float acc[NR][MATS][4];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const float2 lo = unpack(acc2[n][m][0]), hi = unpack(acc2[n][m][1]);
          acc[n][m][0] = lo.x; acc[n][m][1] = lo.y; acc[n][m][2] = hi.x; acc[n][m][3] = hi.y;
        }
      // lanes of a warp that hold the same columns
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[n][m][c] += __shfl_xor_sync(0xffffffffu, acc[n][m][c], o);
      // Sums of the warps, four rows at a time; each goes to the inbox of the block that finishes its columns:
      // inbox[item parity][from][n][m][CPW / S columns].  The place is free: whoever sends item i + 2 has received every
      // block's item i + 1, which each sent after it had read item i.
      constexpr int CV = CPW / 4, OV = CV / S;        // vectors per row of the item, and per owner
      const uint32_t par = done & 1u, inbox = box + par * Cfg::BOX_BYTES;
      if (threadIdx.x == 0) mbar_arrive_expect_tx(smem_u32(&bar_box[par]), Cfg::BOX_BYTES);
#pragma unroll
      for (int g = 0; g < NR; g += Cfg::GROUP) {
        if (lane < LPR) {
#pragma unroll
          for (int n = 0; n < Cfg::GROUP; ++n)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
              sts_v4(red + (((warp * Cfg::GROUP + n) * MATS + m) * CV + lane) * 16,
                     make_float4(acc[g + n][m][0], acc[g + n][m][1], acc[g + n][m][2], acc[g + n][m][3]));
        }
        workers_sync();
        if (g == 0 && lost[0]) {
          alive = false;
          break;
        }
        for (int e = threadIdx.x; e < Cfg::GROUP * MATS * CV; e += ROWS_WORKERS) {
          float4 v = lds_v4(red + e * 16);
#pragma unroll
          for (int w = 1; w < ROWS_WARPS; ++w) {
            const float4 u = lds_v4(red + (w * Cfg::GROUP * MATS * CV + e) * 16);
            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
          }
          const int nm = g * MATS + e / CV, c = e % CV;       // (n * MATS + m), vector of the row
          const uint32_t owner = c / OV;
          const uint32_t at = inbox + ((rank * NR * MATS + nm) * OV + c % OV) * 16;
          const uint32_t bar = smem_u32(&bar_box[par]);
          if (S == 1) st_async_v4(mapa(at, 0u), v, mapa(bar, 0u));
          else st_async_v4(mapa(at, owner), v, mapa(bar, owner));
        }
        workers_sync();
      }
      if (!alive) break;
      if (loses == ROWS_WARPS || !mbar_wait(smem_u32(&bar_box[par]), (done >> 1) & 1u, &abort_flag)) {
        if (lane == 0) give_up(ROLE_ROWS_SUM, item);
        lost[1] = 1;
        workers_sync();
        break;
      }
      for (int e = threadIdx.x; e < NR * OV; e += ROWS_WORKERS) {
        const int n = e / OV, c = e % OV;
        const int col = item * CPW + (static_cast<int>(rank) * OV + c) * 4;
        float v[MATS * 4];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int r = 0; r < S; ++r) {
            const float4 u = lds_v4(inbox + ((r * NR * MATS + n * MATS + m) * OV + c) * 16);
            a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
          }
          v[m * 4] = a.x; v[m * 4 + 1] = a.y; v[m * 4 + 2] = a.z; v[m * 4 + 3] = a.w;
        }
        if (n < p.N && col < p.M) {          // M is a multiple of 4
          const long long at = static_cast<long long>(n) * p.M + col;
          if constexpr (MATS == 2) {
            if (p.G != nullptr) {
              *reinterpret_cast<float4*>(p.G + at) = make_float4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<float4*>(p.U + at) = make_float4(v[4], v[5], v[6], v[7]);
            }
            gated_forward<4>(p.act, v);
          }
          *reinterpret_cast<float4*>(p.out + at) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
      workers_sync();                        // the inbox has been read before this block sends its next item
      if (lost[1]) break;
    }
  }
  __syncthreads();
  if (abort_flag) linger();
  if (S > 1) cluster_sync();                 // nobody leaves while a block may still send to it
}

// 2-D map without swizzle: rows of `inner` floats, boxes of b1 rows x b0 floats, zeros outside.
int make_map_rows(CUtensorMap* m, const float* base, uint64_t inner, uint64_t rows, uint32_t b0, uint32_t b1) {
  return make_map3_as(m, base, inner, rows, 1, inner, inner * rows, b0, b1, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Clusters of S blocks that run at the same time (asked once per device and kernel).
template <int NR, int MATS, int CPW, int S>
cudaError_t rows_clusters(int* count) {
  using Cfg = RowsCfg<NR, MATS, CPW, S>;
  auto kernel = rows_kernel<NR, MATS, CPW, S>;
  static std::atomic<int> cache[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  *count = cache[dev & 63].load(std::memory_order_acquire);
  if (*count > 0) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t q = {};
  q.gridDim = dim3(static_cast<unsigned>(device_sm_count() / S * S), 1, 1);
  q.blockDim = dim3(ROWS_THREADS, 1, 1);
  q.dynamicSmemBytes = Cfg::SMEM;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  q.attrs = attr;
  q.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(count, kernel, &q);
  if (e != cudaSuccess) return e;
  if (*count < 1) return cudaErrorLaunchOutOfResources;
  cache[dev & 63].store(*count, std::memory_order_release);
  return cudaSuccess;
}

struct RowsCall {
  const float* X; const float* W0; const float* W1;
  float* out; float* G; float* U;
  int N, M, K, act, early;
};

template <int NR, int MATS, int CPW, int S>
int rows_launch(const RowsCall& c, cudaStream_t st) {
  using Cfg = RowsCfg<NR, MATS, CPW, S>;
  RowsParams p;
  std::memset(&p, 0, sizeof(p));
  if (int rc = make_map_rows(&p.tmW[0], c.W0, c.M, c.K, CPW, Cfg::KT)) return rc;
  if (MATS == 2)
    if (int rc = make_map_rows(&p.tmW[1], c.W1, c.M, c.K, CPW, Cfg::KT)) return rc;
  if (int rc = make_map_rows(&p.tmX, c.X, c.K, c.N, Cfg::KT, NR)) return rc;
  p.out = c.out; p.G = c.G; p.U = c.U;
  p.N = c.N; p.M = c.M; p.act = c.act; p.early = c.early; p.give_up = rows_give_up();
  p.ktiles = (c.K + Cfg::KT - 1) / Cfg::KT;
  p.items = (c.M + CPW - 1) / CPW;
  cudaError_t e = rows_clusters<NR, MATS, CPW, S>(&p.clusters);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (p.clusters > p.items) p.clusters = p.items;
  p.status = status_word_ptr(&e);
  if (!p.status) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.clusters) * S, 1, 1);
  cfg.blockDim = dim3(ROWS_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c.early ? 2 : 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, rows_kernel<NR, MATS, CPW, S>, p));
}

// Columns per item and blocks per cluster: what a block has to read (its items' tiles) decides, at 30 KB more per item for
// the sums' way to their owner; on equal terms the wider columns (longer runs in memory).  Clusters of two use every SM;
// clusters of four leave about a tenth idle (33 fit on 148 SMs).
template <int NR, int MATS>
int rows_shape(const RowsCall& c, cudaStream_t st) {
  const int sms = device_sm_count();
  int best_w = 128, best_s = 1;
  double best = 1e300;
  for (int w = 128; w >= 32; w >>= 1)
    for (int s = 1; s <= 4; s <<= 1) {
      const int ktiles = static_cast<int>((static_cast<long long>(c.K) * w + 4095) / 4096);
      if (ktiles < s) continue;
      const int items = (c.M + w - 1) / w, clusters = s == 4 ? sms * 2 / 9 : sms / s;
      const double rounds = (items + clusters - 1) / clusters;
      const double cost = rounds * (((ktiles + s - 1) / s) * MATS * 16384.0 + 30e3);
      if (cost < best * 0.97) { best = cost; best_w = w; best_s = s; }
    }
  switch (best_w * 8 + best_s) {
    case 128 * 8 + 1: return rows_launch<NR, MATS, 128, 1>(c, st);
    case 128 * 8 + 2: return rows_launch<NR, MATS, 128, 2>(c, st);
    case 128 * 8 + 4: return rows_launch<NR, MATS, 128, 4>(c, st);
    case 64 * 8 + 1: return rows_launch<NR, MATS, 64, 1>(c, st);
    case 64 * 8 + 2: return rows_launch<NR, MATS, 64, 2>(c, st);
    case 64 * 8 + 4: return rows_launch<NR, MATS, 64, 4>(c, st);
    case 32 * 8 + 1: return rows_launch<NR, MATS, 32, 1>(c, st);
    case 32 * 8 + 2: return rows_launch<NR, MATS, 32, 2>(c, st);
    default: return rows_launch<NR, MATS, 32, 4>(c, st);
  }
}

constexpr int ROWS_MAX = 8;

template <int MATS>
int rows_any(const RowsCall& c, cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  if (c.N <= 1) return rows_shape<1, MATS>(c, st);
  if (c.N <= 2) return rows_shape<2, MATS>(c, st);
  if (c.N <= 4) return rows_shape<4, MATS>(c, st);
  return rows_shape<8, MATS>(c, st);
}

// ------------------------------------------------------------------ many rows
// Estimated time in seconds of an [M, N] product over nkb k-blocks cut into gz slices, on the given tile: waves over
// the SMs x a tile's k-blocks at the measured FP32-accurate rate of that tile (TFLOP/s with every SM busy, the table of
// the plain contraction), a start-up per launch, and for gz > 1 the summation's launch and traffic.
double tile_time(int tile, long long M, long long N, int nkb, int gz) {
  static const double rate[TILE_COUNT] = {118.0, 170.0, 190.0, 206.0, 278.0, 105.0};
  const double sms = device_sm_count();
  const int ctas = tile_ctas(tile), bn = tile_bn(tile);
  const double n_cta = static_cast<double>((M + 128 * ctas - 1) / (128 * ctas)) * static_cast<double>((N + bn - 1) / bn) * ctas * gz;
  const double waves = static_cast<double>(static_cast<long long>((n_cta + sms - 1.0) / sms));
  const double per_cta = static_cast<double>((nkb + gz - 1) / gz) * (2.0 * 128 * bn * 32) / (rate[tile] * 1e12 / 148.0);
  double t = waves * per_cta + 4e-6;
  if (gz > 1) t += 3e-6 + (gz + 1.0) * static_cast<double>(M) * static_cast<double>(N) * 4.0 / 5e12;
  return t;
}

int best_tile(const int* tiles, int count, long long M, long long N, int nkb, int gz, double* time) {
  int best = tiles[0];
  double best_t = 1e300;
  const int forced = forced_tile();      // the "tile" tuning key, where this form has that tile
  for (int i = 0; i < count; ++i) {
    if (tiles[i] == forced) {
      if (time) *time = tile_time(forced, M, N, nkb, gz);
      return forced;
    }
  }
  for (int i = 0; i < count; ++i) {
    const double t = tile_time(tiles[i], M, N, nkb, gz);
    if (t < best_t) { best_t = t; best = tiles[i]; }
  }
  if (time) *time = best_t;
  return best;
}

const int GATED_TILES[3] = {TILE_1x128, TILE_2x128, TILE_2x256};
const int DUAL_TILES[4] = {TILE_1x64, TILE_1x128, TILE_2x128, TILE_2x256};
const int PLAIN_TILES[6] = {TILE_1x64, TILE_1x128, TILE_1x256, TILE_2x128, TILE_2x256, TILE_2x64};

// Slices of the reduction for an [M, N] product when `room` floats of partial sums are at hand.
int split_of(const int* tiles, int count, long long M, long long N, int nkb, long long room, double uncut = 1e300) {
  int best = 1;
  double best_t = uncut;      // what the product takes in one piece by another plan, where there is one
  for (int gz = 1; gz <= 16; ++gz) {
    if (gz > 1 && (nkb / gz < 4 || (gz - 1) * M * N > room)) break;
    double t;
    best_tile(tiles, count, M, N, nkb, gz, &t);
    if (t < best_t) { best_t = t; best = gz; }
  }
  return best;
}

int sum_slices(int64_t stream, float* C, const float* Cbuf, int gz, long long size) {
  return gz > 1 ? cu32_SKbuf_summary(stream, Cbuf, C, gz - 1, static_cast<int>(size)) : CU32_OK;
}

// A launch covers its columns in one piece, or in two: as many columns as fill whole rounds of 256x256 tiles on the
// machine, and the rest in smaller tiles beside the last round (172 tiles are 2.3 rounds of 74 pairs: three rounds, or two
// and a half-size one).  per_unit: tile columns per output column (the gated form's tile holds two per hidden unit).
struct ColumnPlan { int first_cols, first_tile, rest_tile; double time; };

ColumnPlan plan_columns(const int* tiles, int count, long long M, int N, int nkb, int per_unit) {
  ColumnPlan best{};
  double best_t;
  best.first_cols = N;
  best.first_tile = best_tile(tiles, count, M, static_cast<long long>(N) * per_unit, nkb, 1, &best_t);
  best.time = best_t;
  if (forced_tile() >= 0) return best;
  const int unit = 256 / per_unit;
  const long long tiles_m = (M + 255) / 256, pairs = device_sm_count() / 2;
  for (long long rounds = 1; rounds * pairs / tiles_m * unit < N; ++rounds) {
    const int cols = static_cast<int>(rounds * pairs / tiles_m) * unit;
    if (cols <= 0) continue;
    double rest_t;
    const int rest = best_tile(tiles, count, M, static_cast<long long>(N - cols) * per_unit, nkb, 1, &rest_t);
    const double t = tile_time(TILE_2x256, M, static_cast<long long>(cols) * per_unit, nkb, 1) + rest_t - 2e-6;
    if (t < 0.97 * best_t) { best_t = t; best = ColumnPlan{cols, TILE_2x256, rest, t}; }
  }
  return best;
}

// Where a launch stands to the one before it on the stream.
enum Order {
  AFTER,       // behind it entirely: the first launch of a call
  BEHIND,      // depends on it, a launch of the same call: only the start-up overlaps its end
  BESIDE,      // may share the machine with it (whose last tiles leave SMs idle): it neither writes what this one reads nor
               // reads what it writes, and has itself waited for whatever this one depends on
};

// C[M,N] = op(A) op(B) through the plain contraction, cut along K or along its columns where that pays.  A product cut along
// K is never BESIDE the previous launch (the scratch is one).
int product(const int64_t* s, bool a_mn, bool b_mn, const float* A, long long lda, const float* B, long long ldb, float* C,
            int M, int N, int K, float* work, long long room, cudaStream_t st, Order order) {
  GemmCall c{};
  c.A = A; c.B = B; c.C = C; c.Cbuf = work;
  c.M = M; c.N = N; c.K = K; c.n_store = N;
  c.lda = lda; c.ldb = ldb; c.ldc = N; c.a_mn = a_mn; c.b_mn = b_mn;
  c.batch = 1; c.sC = static_cast<long long>(M) * N;
  const int nkb = (K + 31) / 32;
  const ColumnPlan plan = plan_columns(PLAIN_TILES, 6, M, N, nkb, 1);
  c.gz = split_of(PLAIN_TILES, 6, M, N, nkb, work ? room : 0, plan.time);
  c.x3 = true; c.stream = st; c.kc = GATED_KC;
  c.beside_prev = order == BESIDE && c.gz == 1;
  c.behind_prev = order != AFTER;
  if (c.gz > 1) {
    if (int rc = run_gemm(c)) return rc;
    return sum_slices(s[0], C, work, c.gz, c.sC);
  }
  c.N = c.n_store = plan.first_cols;
  if (int rc = run_gemm(c)) return rc;
  if (plan.first_cols == N) return CU32_OK;
  note_column_cut();
  c.B = b_mn ? B + plan.first_cols : B + plan.first_cols * ldb;
  c.C = C + plan.first_cols;
  c.N = c.n_store = N - plan.first_cols;
  c.beside_prev = true;
  return run_gemm(c);
}

// What every launch of the contraction kernel needs besides its operand maps.
int fill_common(GemmParams* p, int M, int N, int nkb, int tile, int out_bn) {
  p->M = M; p->N = N; p->ldc = N;
  p->nkb_total = nkb;
  p->tiles_m = (M + 128 * tile_ctas(tile) - 1) / (128 * tile_ctas(tile));
  p->tiles_n = (N + out_bn - 1) / out_bn;
  p->gz = 1;
  p->kc = GATED_KC;
  choose_rings(p);
  p->vec4_ok = 1;
  cudaError_t e;
  p->status = status_word_ptr(&e);
  return p->status ? CU32_OK : static_cast<int>(e);
}

// H = act(X Wg) * (X Wu) on the tensor cores, G and U stored when G is not null: columns [c0, c0 + cols).
int gated_part(const float* X, const float* Wg, const float* Wu, float* G, float* U, float* H, int N, int D, int F, int act,
               int c0, int cols, int tile, bool beside, cudaStream_t st) {
  const int nkb = (D + 31) / 32;
  note_tile(tile);
  GemmParams p;
  std::memset(&p, 0, sizeof(p));
  const uint64_t n = N, d = D, f = F, w = cols;
  if (int rc = make_map3(&p.tmA, X, d, n, 1, d, d * n, 32, 128, false)) return rc;
  if (int rc = make_map3(&p.tmB, Wg + c0, w, d, 1, f, f * d, 32, 32, true)) return rc;
  if (int rc = make_map3(&p.tmRep[3], Wu + c0, w, d, 1, f, f * d, 32, 32, true)) return rc;
  if (int rc = make_map3(&p.tmC, H + c0, w, n, 1, f, f * n, 32, 32, false)) return rc;
  if (G) {
    if (int rc = make_map3(&p.tmRep[0], G + c0, w, n, 1, f, f * n, 32, 32, false)) return rc;
    if (int rc = make_map3(&p.tmRep[1], U + c0, w, n, 1, f, f * n, 32, 32, false)) return rc;
    p.gated_save = 1;
  }
  if (int rc = fill_common(&p, N, cols, nkb, tile, tile_bn(tile) / 2)) return rc;
  p.C = H + c0; p.ldc = F; p.act = act; p.tma_store = 1;
  p.overlap_prev = p.join_prev = beside ? 1 : 0;
  // One flush: the activation needs the complete sums.  Beyond D = 8192, where plain products put their registers' sums down
  // in memory, these chains of D / 32 additions go on: 3.6e-7 off at D = 8192, 4.7e-7 at 16384, 8.3e-7 at 65536.
  p.flush_chunks = nkb;
  return static_cast<int>(launch_gemm_gated(tile, p, st));
}

int gated_tiles(const float* X, const float* Wg, const float* Wu, float* G, float* U, float* H, int N, int D, int F, int act,
                cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  const ColumnPlan c = plan_columns(GATED_TILES, 3, N, F, (D + 31) / 32, 2);
  if (int rc = gated_part(X, Wg, Wu, G, U, H, N, D, F, act, 0, c.first_cols, c.first_tile, false, st)) return rc;
  if (c.first_cols == F) return CU32_OK;
  note_column_cut();
  return gated_part(X, Wg, Wu, G, U, H, N, D, F, act, c.first_cols, F - c.first_cols, c.rest_tile, true, st);
}

// deltaG = deltaH * U * act'(G) and deltaU = deltaH * act(G), deltaH read where deltaG is written.  A pass of its own
// (five floats per element, 36 us for 2048 x 5464): as the epilogue of deltaH's product it took more than it saved,
// because a tile's epilogue stands in the way of the next tile's products (two rounds of K = 2048 tiles: 135 us as
// straight-line code, waiting for instructions; 102 us as a loop; 64 us for the plain product).
// Each thread reads its elements before it writes them, so deltaU may lie over G or U.
__global__ void __launch_bounds__(256) gated_delta_kernel(float* dG, float* dU, const float* G, const float* U, long long vecs,
                                                          int act) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long v = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; v < vecs; v += 2 * stride) {
    const bool two = v + stride < vecs;
    const long long w = two ? v + stride : v;
    const float4 d0 = reinterpret_cast<const float4*>(dG)[v], g0 = reinterpret_cast<const float4*>(G)[v],
                 u0 = reinterpret_cast<const float4*>(U)[v];
    const float4 d1 = reinterpret_cast<const float4*>(dG)[w], g1 = reinterpret_cast<const float4*>(G)[w],
                 u1 = reinterpret_cast<const float4*>(U)[w];
    float4 a, b;
    gated_backward4(act, d0, g0, u0, &a, &b);
    reinterpret_cast<float4*>(dG)[v] = a;
    reinterpret_cast<float4*>(dU)[v] = b;
    if (two) {
      gated_backward4(act, d1, g1, u1, &a, &b);
      reinterpret_cast<float4*>(dG)[w] = a;
      reinterpret_cast<float4*>(dU)[w] = b;
    }
  }
}

// deltaX = deltaG Wg^T + deltaU Wu^T
int dual_tiles(const int64_t* s, const float* dG, const float* Wg, const float* dU, const float* Wu, float* dX, int N, int D,
               int F, float* work, long long room, cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  const int half = (F + 31) / 32;
  const int gz = split_of(DUAL_TILES, 4, N, D, 2 * half, work ? room : 0);
  const int tile = note_tile(best_tile(DUAL_TILES, 4, N, D, 2 * half, gz, nullptr));
  GemmParams p;
  std::memset(&p, 0, sizeof(p));
  const uint64_t n = N, d = D, f = F;
  const uint32_t bbox = tile_bn(tile) / tile_ctas(tile);
  p.overlap_prev = p.wait_prev = 1;      // behind what wrote dG and dU
  if (int rc = make_map3(&p.tmA, dG, f, n, 1, f, f * n, 32, 128, false)) return rc;
  if (int rc = make_map3(&p.tmRep[2], dU, f, n, 1, f, f * n, 32, 128, false)) return rc;
  if (int rc = make_map3(&p.tmB, Wg, f, d, 1, f, f * d, 32, bbox, false)) return rc;
  if (int rc = make_map3(&p.tmRep[3], Wu, f, d, 1, f, f * d, 32, bbox, false)) return rc;
  if (int rc = make_map3(&p.tmC, dX, d, n, 1, d, d * n, 32, 32, false)) return rc;
  if (gz > 1)
    if (int rc = make_map3(&p.tmCbuf, work, d, n, gz - 1, d, d * n, 32, 32, false)) return rc;
  if (int rc = fill_common(&p, N, D, 2 * half, tile, tile_bn(tile))) return rc;
  p.C = dX; p.Cbuf = work; p.c_stride = static_cast<long long>(N) * D;
  p.gz = gz; p.tma_store = 1; p.nkb_first = half;
  if (cudaError_t e = launch_gemm_dual(tile, p, gz, st)) return static_cast<int>(e);
  return sum_slices(s[0], dX, work, gz, p.c_stride);
}

int check_dims(int N, int D, int F, int act) {
  if (N <= 0 || D <= 0 || F <= 0) return CU32_E_DIM;
  if (static_cast<long long>(N) * D >= (1LL << 31) || static_cast<long long>(N) * F >= (1LL << 31) ||
      static_cast<long long>(D) * F >= (1LL << 31))
    return CU32_E_DIM;
  if (act < CU32_ACT_SILU || act > CU32_ACT_SIGMOID) return CU32_E_ARG;
  if ((D & 3) || (F & 3)) return CU32_E_ALIGN;
  return CU32_OK;
}

long long thin_floats(int N, int D, int F) {
  const long long up = thin_work_floats(N, F, D, THIN_GATED), down = thin_work_floats(N, D, F, THIN_PLAIN);
  return up > down ? up : down;
}
long long thin_delta_floats(int N, int D, int F) {
  const long long h = thin_work_floats(N, F, D, THIN_DELTA), x = thin_work_floats(N, D, F, THIN_DUAL);
  return h > x ? h : x;
}

template <class... P>
bool any_null(const P*... p) { return (... || (p == nullptr)); }
template <class... P>
bool all_aligned16(const P*... p) { return (... && aligned16(p)); }

// An array of a call; null where the call neither reads nor writes it.
struct Span { const float* p; long long n; };
inline bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.p && b.p && x < y + 4ull * static_cast<unsigned long long>(b.n) && y < x + 4ull * static_cast<unsigned long long>(a.n);
}
// Whether an output lies over an operand or another output.  Which of them would still come out right depends on the form a
// call takes, and so on the number of rows: all are refused.
template <int OUTS, int INS>
bool outputs_overlap(const Span (&out)[OUTS], const Span (&in)[INS]) {
  for (int i = 0; i < OUTS; ++i) {
    for (int j = 0; j < INS; ++j)
      if (overlap(out[i], in[j])) return true;
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return true;
  }
  return false;
}

}  // namespace
}  // namespace dragon

using namespace dragon;

extern "C" {

long long cu32_gatedFF_work(int N, int D, int F) {
  if (check_dims(N, D, F, CU32_ACT_SILU)) return 0;
  const long long any = 1LL << 60;
  const long long n = N, d = D, f = F;
  auto extra = [](int gz, long long size) { return (gz - 1) * size; };
  const long long a = extra(split_of(PLAIN_TILES, 6, n, d, (F + 31) / 32, any), n * d);       // Y
  const long long b = extra(split_of(DUAL_TILES, 4, n, d, 2 * ((F + 31) / 32), any), n * d);  // deltaX
  const long long c = extra(split_of(PLAIN_TILES, 6, d, f, (N + 31) / 32, any), d * f);       // deltaWg, deltaWu
  const long long e = extra(split_of(PLAIN_TILES, 6, f, d, (N + 31) / 32, any), d * f);       // deltaWd
  const long long h = extra(split_of(PLAIN_TILES, 6, n, f, (D + 31) / 32, any), n * f);       // deltaH
  long long most = a;
  for (const long long x : {b, c, e, h})
    if (x > most) most = x;
  if (N > THIN_MAX_ROWS) return most;
  const long long forward = N > ROWS_MAX ? thin_floats(N, D, F) : 0, backward = thin_delta_floats(N, D, F);
  if (forward > most) most = forward;
  return backward > most ? backward : most;
}

int cu32_gatedFF(const int64_t* s, int length, const float* X, const float* Wg, const float* Wu, const float* Wd, float* G,
                 float* U, float* H, float* Y, float* work, long long work_floats, int N, int D, int F, int act) {
  load_env_once();
  cudaStream_t st;
  if (int rc = check_streams(s, length, &st)) return rc;
  if (any_null(X, Wg, Wu, Wd, H, Y) || (G == nullptr) != (U == nullptr)) return CU32_E_NULL;
  if (int rc = check_dims(N, D, F, act)) return rc;
  if (!all_aligned16(X, Wg, Wu, Wd, G, U, H, Y, work)) return CU32_E_ALIGN;
  const long long nd = static_cast<long long>(N) * D, nf = static_cast<long long>(N) * F, df = static_cast<long long>(D) * F;
  if (outputs_overlap({{G, nf}, {U, nf}, {H, nf}, {Y, nd}}, {{X, nd}, {Wg, df}, {Wu, df}, {Wd, df}})) return CU32_E_ARG;
  if (N <= ROWS_MAX) {
    const RowsCall up{X, Wg, Wu, H, G, U, N, F, D, act, 0};
    if (int rc = rows_any<2>(up, st)) return rc;
    const RowsCall down{H, Wd, nullptr, Y, nullptr, nullptr, N, D, F, 0, 1};
    return rows_any<1>(down, st);
  }
  if (N <= THIN_MAX_ROWS && work && thin_floats(N, D, F) <= work_floats) {
    const ThinCall up{X, nullptr, Wg, Wu, H, G, U, nullptr, nullptr, work, N, F, D, act, 0};
    if (int rc = thin_product(up, THIN_GATED, st)) return rc;
    const ThinCall down{H, nullptr, Wd, nullptr, Y, nullptr, nullptr, nullptr, nullptr, work, N, D, F, 0, 1};
    return thin_product(down, THIN_PLAIN, st);
  }
  if (int rc = gated_tiles(X, Wg, Wu, G, U, H, N, D, F, act, st)) return rc;
  return product(s, false, true, H, F, Wd, D, Y, N, D, F, work, work_floats, st, BEHIND);
}

int cu32_gatedFF_delta(const int64_t* s, int length, const float* dY, const float* X, const float* Wg, const float* Wu,
                       const float* Wd, const float* G, const float* U, const float* H, float* dG, float* dU, float* dX,
                       float* dWg, float* dWu, float* dWd, float* work, long long work_floats, int N, int D, int F, int act) {
  load_env_once();
  cudaStream_t st;
  if (int rc = check_streams(s, length, &st)) return rc;
  if (any_null(dY, Wd, G, U, dG, dU)) return CU32_E_NULL;
  if (dG == G || dG == U || dG == dU) return CU32_E_ARG;      // deltaH is formed where deltaG will be
  if ((dX && any_null(Wg, Wu)) || ((dWg || dWu) && !X) || (dWd && !H)) return CU32_E_NULL;
  if (int rc = check_dims(N, D, F, act)) return rc;
  if (!all_aligned16(dY, X, Wg, Wu, Wd, G, U, H, dG, dU, dX, dWg, dWu, dWd, work)) return CU32_E_ALIGN;
  const long long nd = static_cast<long long>(N) * D, nf = static_cast<long long>(N) * F, df = static_cast<long long>(D) * F;
  const float* const x = dWg || dWu ? X : nullptr;      // operands that only some of the gradients need
  const float* const h = dWd && H != dG ? H : nullptr;  // and those that are replaced
  const float *const g = G != dU ? G : nullptr, *const u = U != dU ? U : nullptr;
  if (outputs_overlap({{dG, nf}, {dU, nf}, {dX, nd}, {dWg, df}, {dWu, df}, {dWd, df}},
                      {{dY, nd}, {x, nd}, {dX ? Wg : nullptr, df}, {dX ? Wu : nullptr, df}, {Wd, df}, {g, nf}, {u, nf}, {h, nf}}))
    return CU32_E_ARG;
  // Launches that do not depend on each other stand side by side, so that the tiles of the next fill the last round of
  // the one before: deltaWd with deltaH, and deltaWg with deltaWu.  With few rows all three are one launch at the end
  // (deltaWd, which reads H, before the others where deltaG replaces H).
  const bool outer = N <= OUTER_MAX_ROWS, first = dWd && (!outer || dG == H);
  const OuterPair of_down{H, dY, dWd, F, D};
  if (first && outer) {
    if (int rc = outer_products(&of_down, 1, N, false, st)) return rc;
  } else if (first) {
    if (int rc = product(s, true, true, H, F, dY, D, dWd, F, D, N, work, work_floats, st, AFTER)) return rc;
  }
  if (N <= THIN_MAX_ROWS && work && thin_delta_floats(N, D, F) <= work_floats) {
    const ThinCall h{dY, nullptr, Wd, nullptr, dG, nullptr, dU, G, U, work, N, F, D, act, first};
    if (int rc = thin_product(h, THIN_DELTA, st)) return rc;
    if (dX) {
      const ThinCall x{dG, dU, Wg, Wu, dX, nullptr, nullptr, nullptr, nullptr, work, N, D, F, 0, 1};
      if (int rc = thin_product(x, THIN_DUAL, st)) return rc;
    }
  } else {
    const Order order = !first ? AFTER : dG == H ? BEHIND : BESIDE;
    if (int rc = product(s, false, false, dY, D, Wd, D, dG, N, F, D, work, work_floats, st, order)) return rc;
    const long long vecs = static_cast<long long>(N) * F / 4;
    long long blocks = (vecs + 511) / 512;
    if (blocks > 16LL * device_sm_count()) blocks = 16LL * device_sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, gated_delta_kernel, dG, dU, G, U, vecs, act)) return static_cast<int>(e);
    if (dX)
      if (int rc = dual_tiles(s, dG, Wg, dU, Wu, dX, N, D, F, work, work_floats, st)) return rc;
  }
  if (outer) {
    OuterPair pairs[3];
    int count = 0;
    if (dWg) pairs[count++] = OuterPair{X, dG, dWg, D, F};
    if (dWu) pairs[count++] = OuterPair{X, dU, dWu, D, F};
    if (dWd && !first) pairs[count++] = of_down;
    return count > 0 ? outer_products(pairs, count, N, true, st) : CU32_OK;
  }
  if (dWg)
    if (int rc = product(s, true, true, X, D, dG, F, dWg, D, F, N, work, work_floats, st, BEHIND)) return rc;
  if (dWu)
    if (int rc = product(s, true, true, X, D, dU, F, dWu, D, F, N, work, work_floats, st, dWg ? BESIDE : BEHIND)) return rc;
  return CU32_OK;
}

}  // extern "C"
