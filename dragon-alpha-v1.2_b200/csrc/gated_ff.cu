// Gated feed-forward block:  H = act(X Wg) * (X Wu),  Y = H Wd,  and its gradients.
//
//   X [N, D], Wg, Wu [D, F], Wd [F, D]; G = X Wg, U = X Wu.
//   deltaH = deltaY Wd^T;  deltaG = deltaH * U * act'(G);  deltaU = deltaH * act(G)
//   deltaX = deltaG Wg^T + deltaU Wu^T;  deltaWg = X^T deltaG;  deltaWu = X^T deltaU;  deltaWd = H^T deltaY
//
// Many rows: the contraction kernel (gemm_tf32.cuh) with three epilogues of its own - both projections in one launch
// with act(G) * U formed in the registers that hold the sums, deltaH turned into deltaG and deltaU before it is stored,
// and the two products of deltaX in one accumulation.  6 N D F flop forward and 12 N D F backward at the
// FP32-accurate rate bound it.
// Few rows: every weight is read once for all rows, so the time is that of reading 3 D F floats; rows_kernel below.
#include <cooperative_groups.h>
#include <atomic>

#include "cu32_host.h"

namespace dragon {
namespace {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ few rows
struct RowsParams {
  const float* X;             // [N, K]
  const float* W[2];          // [K, M]; the second only for the gated form
  float* out;                 // [N, M]
  float* G;                   // gated form: pre-activations, or null
  float* U;
  int N, M, K, act;
  int kc;                     // rows of K staged at a time
};

__device__ __forceinline__ float4 ldg_stream(const float* p) {
  float4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

constexpr int ROWS_THREADS = 256, ROWS_WARPS = ROWS_THREADS / 32;

// out[n, :] = X[n, :] W  (MATS = 1)  or  act(X[n, :] W0) * (X[n, :] W1)  (MATS = 2)  for N <= NR rows.
// A cluster owns CPW columns and its CTAs a slice of K each; inside a CTA the warps take every eighth (group of) row(s)
// of the weights, 16 bytes per lane.  X's slice sits in shared memory as [k][NR], so one broadcast read serves four rows.
// The partial sums of lanes, warps and CTAs are added in a fixed order: results do not vary from run to run.
template <int NR, int MATS, int CPW>
__global__ void __launch_bounds__(ROWS_THREADS) rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ float4 rows_smem4[];
  float* sm = reinterpret_cast<float*>(rows_smem4);
  cg::cluster_group cluster = cg::this_cluster();
  const int S = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  constexpr int LPR = CPW / 4, KPW = 32 / LPR, STEP = ROWS_WARPS * KPW;
  constexpr int UN = MATS == 2 ? 4 : 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col0 = (blockIdx.x / S) * CPW;
  const int col = col0 + (lane % LPR) * 4;
  const bool col_ok = col < p.M;    // M is a multiple of 4
  const int k0 = static_cast<int>(static_cast<long long>(rank) * p.K / S);
  const int k1 = static_cast<int>(static_cast<long long>(rank + 1) * p.K / S);
  float acc[NR][MATS][4];
#pragma unroll
  for (int n = 0; n < NR; ++n)
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][m][c] = 0.0f;

  for (int kb = k0; kb < k1; kb += p.kc) {
    const int ke = min(kb + p.kc, k1);
    __syncthreads();                      // the previous slice has been read
    for (int i = threadIdx.x; i < (ke - kb) * NR; i += ROWS_THREADS) {
      const int n = i / (ke - kb), k = i - n * (ke - kb);
      sm[k * NR + n] = n < p.N ? p.X[static_cast<long long>(n) * p.K + kb + k] : 0.0f;
    }
    __syncthreads();
    for (int k = kb + warp * KPW + lane / LPR; k < ke; k += STEP * UN) {
      float4 w[UN][MATS];
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const int kk = k + u * STEP;
          w[u][m] = (kk < ke && col_ok) ? ldg_stream(p.W[m] + static_cast<long long>(kk) * p.M + col)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int kk = min(k + u * STEP, ke - 1);
        const float* x = sm + (kk - kb) * NR;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float xv = x[n];
#pragma unroll
          for (int m = 0; m < MATS; ++m) {
            acc[n][m][0] = fmaf(xv, w[u][m].x, acc[n][m][0]);
            acc[n][m][1] = fmaf(xv, w[u][m].y, acc[n][m][1]);
            acc[n][m][2] = fmaf(xv, w[u][m].z, acc[n][m][2]);
            acc[n][m][3] = fmaf(xv, w[u][m].w, acc[n][m][3]);
          }
        }
      }
    }
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
  __syncthreads();
  constexpr int PER = NR * MATS * CPW;    // sums of a CTA: [n][m][column]
  if (lane < LPR) {
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int m = 0; m < MATS; ++m)
        *reinterpret_cast<float4*>(sm + warp * PER + (n * MATS + m) * CPW + lane * 4) =
            make_float4(acc[n][m][0], acc[n][m][1], acc[n][m][2], acc[n][m][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < PER; i += ROWS_THREADS) {
    float s = sm[i];
#pragma unroll
    for (int w = 1; w < ROWS_WARPS; ++w) s += sm[w * PER + i];
    sm[i] = s;
  }
  cluster.sync();
  // the CTAs of the cluster share the outputs: each adds the S partial sums of its part
  for (int i = rank * ROWS_THREADS + threadIdx.x; i < NR * CPW; i += S * ROWS_THREADS) {
    const int n = i / CPW, c = i - n * CPW;
    if (n < p.N && col0 + c < p.M) {
      float v[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        float s = 0.0f;
        for (int r = 0; r < S; ++r) s += cluster.map_shared_rank(sm, r)[(n * MATS + m) * CPW + c];
        v[m] = s;
      }
      const long long at = static_cast<long long>(n) * p.M + col0 + c;
      if (MATS == 2) {
        if (p.G != nullptr) { p.G[at] = v[0]; p.U[at] = v[MATS - 1]; }
        float pair[2] = {v[0], v[MATS - 1]};
        gated_forward<1>(p.act, pair);
        p.out[at] = pair[0];
      } else {
        p.out[at] = v[0];
      }
    }
  }
  cluster.sync();     // nobody leaves while its sums are being read
}

template <int NR, int MATS, int CPW>
int rows_launch_one(RowsParams p, int S, cudaStream_t st) {
  constexpr int SLICE = 16384;            // floats of X staged at a time (64 KB)
  p.kc = SLICE / NR;
  const int klen = (p.K + S - 1) / S;
  if (p.kc > klen) p.kc = klen;
  constexpr int RED = ROWS_WARPS * NR * MATS * CPW;
  const size_t smem = sizeof(float) * static_cast<size_t>(p.kc * NR > RED ? p.kc * NR : RED);
  constexpr size_t MAX_SMEM = sizeof(float) * (SLICE > RED ? SLICE : RED);
  auto kernel = rows_kernel<NR, MATS, CPW>;
  static std::atomic<int> ready[64];      // per device: the shared-memory opt-in has been made
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(MAX_SMEM));
    if (e != cudaSuccess) return static_cast<int>(e);
    ready[dev & 63].store(1, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.M + CPW - 1) / CPW * S), 1, 1);
  cfg.blockDim = dim3(ROWS_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(S);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

// Columns per cluster and CTAs per cluster: wide columns and few slices as long as they give every SM two CTAs.
template <int NR, int MATS>
int rows_launch(const RowsParams& p, cudaStream_t st) {
  const int want = 2 * device_sm_count();
  int cpw = 32, S = 8;
  for (int c = 128; c >= 32 && cpw == 32; c >>= 1) {
    const int blocks = (p.M + c - 1) / c;
    for (int s = 1; s <= 8; s <<= 1)
      if (blocks * s >= want && p.K / s >= 64) { cpw = c; S = s; break; }
    if (cpw != 32 || (c == 32 && blocks * S >= want)) break;
  }
  while (S > 1 && p.K / S < 16) S >>= 1;
  if (cpw == 128) return rows_launch_one<NR, MATS, 128>(p, S, st);
  if (cpw == 64) return rows_launch_one<NR, MATS, 64>(p, S, st);
  return rows_launch_one<NR, MATS, 32>(p, S, st);
}

constexpr int ROWS_MAX = 16;

template <int MATS>
int rows_any(const RowsParams& p, cudaStream_t st) {
  if (p.N <= 1) return rows_launch<1, MATS>(p, st);
  if (p.N <= 2) return rows_launch<2, MATS>(p, st);
  if (p.N <= 4) return rows_launch<4, MATS>(p, st);
  if (p.N <= 8) return rows_launch<8, MATS>(p, st);
  return rows_launch<16, MATS>(p, st);
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
int split_of(const int* tiles, int count, long long M, long long N, int nkb, long long room) {
  static const int cuts[] = {1, 2, 3, 4, 6, 8, 12, 16};
  int best = 1;
  double best_t = 1e300;
  for (int gz : cuts) {
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

// C[M,N] = op(A) op(B) through the plain contraction, cut along K where that pays.
int product(const int64_t* s, bool a_mn, bool b_mn, const float* A, long long lda, const float* B, long long ldb, float* C,
            int M, int N, int K, float* work, long long room, cudaStream_t st) {
  GemmCall c{};
  c.A = A; c.B = B; c.C = C; c.Cbuf = work;
  c.M = M; c.N = N; c.K = K; c.n_store = N;
  c.lda = lda; c.ldb = ldb; c.ldc = N; c.a_mn = a_mn; c.b_mn = b_mn;
  c.batch = 1; c.sC = static_cast<long long>(M) * N;
  c.gz = split_of(PLAIN_TILES, 6, M, N, (K + 31) / 32, work ? room : 0);
  c.x3 = true; c.stream = st;
  if (int rc = run_gemm(c)) return rc;
  return sum_slices(s[0], C, work, c.gz, c.sC);
}

// What every launch of the contraction kernel needs besides its operand maps.
int fill_common(GemmParams* p, int M, int N, int nkb, int tile, int out_bn) {
  p->M = M; p->N = N; p->ldc = N;
  p->nkb_total = nkb;
  p->tiles_m = (M + 128 * tile_ctas(tile) - 1) / (128 * tile_ctas(tile));
  p->tiles_n = (N + out_bn - 1) / out_bn;
  p->gz = 1;
  p->kc = tuned_kc();
  choose_rings(p);
  p->vec4_ok = 1;
  cudaError_t e;
  p->status = status_word_ptr(&e);
  return p->status ? CU32_OK : static_cast<int>(e);
}

// H = act(X Wg) * (X Wu) on the tensor cores, G and U stored when G is not null.
int gated_tiles(const float* X, const float* Wg, const float* Wu, float* G, float* U, float* H, int N, int D, int F, int act,
                cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  const int nkb = (D + 31) / 32;
  const int tile = note_tile(best_tile(GATED_TILES, 3, N, 2LL * F, nkb, 1, nullptr));
  GemmParams p;
  std::memset(&p, 0, sizeof(p));
  const uint64_t n = N, d = D, f = F;
  if (int rc = make_map3(&p.tmA, X, d, n, 1, d, d * n, 32, 128, false)) return rc;
  if (int rc = make_map3(&p.tmB, Wg, f, d, 1, f, f * d, 32, 32, true)) return rc;
  if (int rc = make_map3(&p.tmRep[3], Wu, f, d, 1, f, f * d, 32, 32, true)) return rc;
  if (int rc = make_map3(&p.tmC, H, f, n, 1, f, f * n, 32, 32, false)) return rc;
  if (G) {
    if (int rc = make_map3(&p.tmRep[0], G, f, n, 1, f, f * n, 32, 32, false)) return rc;
    if (int rc = make_map3(&p.tmRep[1], U, f, n, 1, f, f * n, 32, 32, false)) return rc;
    p.gated_save = 1;
  }
  if (int rc = fill_common(&p, N, F, nkb, tile, tile_bn(tile) / 2)) return rc;
  p.C = H; p.act = act; p.tma_store = 1;
  p.flush_chunks = nkb;      // one flush: the activation needs the complete sums
  return static_cast<int>(launch_gemm_gated(tile, p, st));
}

// deltaG, deltaU from deltaY, Wd, G, U.
int dgated_tiles(const float* dY, const float* Wd, const float* G, const float* U, float* dG, float* dU, int N, int D, int F,
                 int act, cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  const int nkb = (D + 31) / 32;
  const int tile = note_tile(best_tile(GATED_TILES, 3, N, F, nkb, 1, nullptr));
  GemmParams p;
  std::memset(&p, 0, sizeof(p));
  const uint64_t n = N, d = D, f = F;
  if (int rc = make_map3(&p.tmA, dY, d, n, 1, d, d * n, 32, 128, false)) return rc;
  if (int rc = make_map3(&p.tmB, Wd, d, f, 1, d, d * f, 32, tile_bn(tile) / tile_ctas(tile), false)) return rc;
  if (int rc = fill_common(&p, N, F, nkb, tile, tile_bn(tile))) return rc;
  p.C = dG; p.act = act;
  p.ep_g = G; p.ep_u = U; p.ep_dg = dG; p.ep_du = dU;
  p.flush_chunks = nkb;
  return static_cast<int>(launch_gemm_dgated(tile, p, st));
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

template <class... P>
bool any_null(const P*... p) { return (... || (p == nullptr)); }
template <class... P>
bool all_aligned16(const P*... p) { return (... && aligned16(p)); }

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
  const long long m = a > b ? a : b, o = c > e ? c : e;
  return m > o ? m : o;
}

int cu32_gatedFF(const int64_t* s, int length, const float* X, const float* Wg, const float* Wu, const float* Wd, float* G,
                 float* U, float* H, float* Y, float* work, long long work_floats, int N, int D, int F, int act) {
  load_env_once();
  cudaStream_t st;
  if (int rc = check_streams(s, length, &st)) return rc;
  if (any_null(X, Wg, Wu, Wd, H, Y) || (G == nullptr) != (U == nullptr)) return CU32_E_NULL;
  if (int rc = check_dims(N, D, F, act)) return rc;
  if (!all_aligned16(X, Wg, Wu, Wd, G, U, H, Y, work)) return CU32_E_ALIGN;
  if (N <= ROWS_MAX) {
    RowsParams p{};
    p.X = X; p.W[0] = Wg; p.W[1] = Wu; p.out = H; p.G = G; p.U = U;
    p.N = N; p.M = F; p.K = D; p.act = act;
    if (int rc = rows_any<2>(p, st)) return rc;
    RowsParams q{};
    q.X = H; q.W[0] = Wd; q.out = Y;
    q.N = N; q.M = D; q.K = F;
    return rows_any<1>(q, st);
  }
  if (int rc = gated_tiles(X, Wg, Wu, G, U, H, N, D, F, act, st)) return rc;
  return product(s, false, true, H, F, Wd, D, Y, N, D, F, work, work_floats, st);
}

int cu32_gatedFF_delta(const int64_t* s, int length, const float* dY, const float* X, const float* Wg, const float* Wu,
                       const float* Wd, const float* G, const float* U, const float* H, float* dG, float* dU, float* dX,
                       float* dWg, float* dWu, float* dWd, float* work, long long work_floats, int N, int D, int F, int act) {
  load_env_once();
  cudaStream_t st;
  if (int rc = check_streams(s, length, &st)) return rc;
  if (any_null(dY, Wd, G, U, dG, dU)) return CU32_E_NULL;
  if ((dX && any_null(Wg, Wu)) || ((dWg || dWu) && !X) || (dWd && !H)) return CU32_E_NULL;
  if (int rc = check_dims(N, D, F, act)) return rc;
  if (!all_aligned16(dY, X, Wg, Wu, Wd, G, U, H, dG, dU, dX, dWg, dWu, dWd, work)) return CU32_E_ALIGN;
  if (dWd)
    if (int rc = product(s, true, true, H, F, dY, D, dWd, F, D, N, work, work_floats, st)) return rc;
  if (int rc = dgated_tiles(dY, Wd, G, U, dG, dU, N, D, F, act, st)) return rc;
  if (dX)
    if (int rc = dual_tiles(s, dG, Wg, dU, Wu, dX, N, D, F, work, work_floats, st)) return rc;
  if (dWg)
    if (int rc = product(s, true, true, X, D, dG, F, dWg, D, F, N, work, work_floats, st)) return rc;
  if (dWu)
    if (int rc = product(s, true, true, X, D, dU, F, dWu, D, F, N, work, work_floats, st)) return rc;
  return CU32_OK;
}

}  // extern "C"
