// Products of a few dozen rows with a large weight, FP32-accurate on the tensor cores:
//   out[n, :] = X[n, :] W   or   act(X[n, :] W0) * (X[n, :] W1),   9 to 128 rows, and for the gradients
//   deltaG, deltaU from deltaH = deltaY W^T,   deltaX = deltaG W0^T + deltaU W1^T,   up to 128 rows.
//
// Every weight is read once for all rows, so the time should be that of reading the weights (with the general kernel it was
// three times that: 315 us for 16 rows of a 4096 / 10924 block, 537 MB).  The roles of the operands
// are therefore exchanged against the general contraction kernel: 128 weight columns are the rows of the tensor core's
// tile (operand A as they lie: MN-major, or K-major for W^T), the NT rows of X its columns - no tile row is wasted on rows
// X does not have.
// Arithmetic as there: hi = what the tensor core makes of an FP32 operand, lo = rounded remainder, written beside it by
// split warps; lo*hi + hi*lo + hi*hi, a stage of the ring summed in tensor memory before FP32 registers take over.
// Up to 64 rows X's lo part lies right behind its hi part, so that one instruction with 2 NT columns forms hi*hi and hi*lo
// and the weight tile is fetched twice per step instead of three times (the fetches from shared memory bound the step).
//
// The work is cut into slices, 128 columns by a share of K, so many that whole rounds of them occupy every SM, and
// numbered with the column block running fastest: what the SMs read at one time are neighbouring columns of the same
// rows.  (Equal runs of a list ordered column block by column block balance better, but read scattered 512-byte pieces:
// 4 TB/s, and asking for them earlier made it slower still.)  A slice's sums go to the caller's scratch and a second kernel
// adds a column block's slices in order, applies the gate and stores the rows (no atomics: results do not vary).
// Measured for a 4096 / 10924 block, forward, in a long graph: 16 rows 119 to 122 us (the reads at 4.8 TB/s), 32 rows 139 to
// 143, 64 rows 168 to 173, 128 rows 264 to 276 us, where X and its parts weigh as much as the weights.
#include <atomic>

#include "cu32_host.h"
#include "gated_thin.h"

namespace dragon {
namespace {

using namespace ptx;

constexpr int THIN_THREADS = 512;
constexpr int ROLE_THIN_LOAD = 13, ROLE_THIN_SPLIT = 14, ROLE_THIN_MMA = 15, ROLE_THIN_DRAIN = 16;

struct ThinParams {
  CUtensorMap tmW[2];       // [K, M] weights, boxes of 32 x 32 (MN-major slabs), or [M, K], boxes of 128 rows x 32
  CUtensorMap tmX[2];       // [N, K], boxes of NT rows x 32 (K-major); the second only for two products in one sum
  int half;                 // two products in one sum: stages of the first, else the number of stages
  float* part;              // [slice][row][128 columns]
  int stages, items, slices, chunk;    // slice id: share of K * items + item; items: column blocks, matrix by matrix;
                                       // K in stages of 32 KS rows, `chunk` of them summed in tensor memory
  int blocks;                          // column blocks of a matrix (items of both matrices at once: as many items)
  int early;                // the grid may start before the one that writes X has ended
  int* status;
};

// MP: matrices per slice.  Up to 32 rows a slice is of one matrix and a stage of the ring holds two blocks of it; beyond, X
// and its split weigh as much as the weights, and a gated slice takes the same block of both matrices against one X.
template <int NT, int MP, bool A_KM = false>
struct ThinCfg {
  static constexpr bool CONCAT = NT <= 64;
  // Rows of 32 per stage of the ring.  What a stage costs whatever its size - the issuing thread's waits and commits, the
  // split's fence - is 700 cycles, the time 16 KB take from memory: two rows of blocks share it where the ring allows.
  static constexpr int KS = NT <= 32 ? 2 : 1;
  static constexpr int SUBS = KS * MP;                            // 16 KB weight tiles of a stage
  static constexpr int W_BYTES = SUBS * 16384;
  static constexpr int X_BYTES = NT * 128;                        // X of 32 rows of K; its lo part behind it
  static constexpr int RAW = W_BYTES + KS * 2 * X_BYTES;
  static constexpr int LO = W_BYTES;                              // lo part of the weights
  // A lo slot is held from the split until the products that read it are seen to be done.
  static constexpr int L = SUBS == 2 ? 2 : 3;
  static constexpr int FIT = (225 * 1024 - L * LO) / RAW;
  static constexpr int R = FIT < 8 ? FIT : 8;
  static constexpr int SMEM = 1024 + R * RAW + L * LO;
  static constexpr int DCOLS = CONCAT ? 2 * NT : NT;              // tensor-memory columns per buffer
  static constexpr int TMEM_NEED = 2 * MP * DCOLS;
  static constexpr int TMEM_COLS = TMEM_NEED <= 64 ? 64 : TMEM_NEED <= 128 ? 128 : TMEM_NEED <= 256 ? 256 : 512;
  // Four drain warps hold all sums of their 32 columns where those are 128 at most, else eight, a matrix each half.  The
  // other warps but two split: all on one stage, or, where a stage is one tile, in two groups that take the stages in turn
  // (a split is mostly latency).
  static constexpr int DRAIN_WARPS = MP * NT <= 128 ? 4 : 8, DRAIN_WARP0 = 16 - DRAIN_WARPS;
  static constexpr int MINE = DRAIN_WARPS == 4 ? MP : 1;          // matrices per drain warp
  static constexpr int GROUPS = SUBS == 2 ? 1 : 2, SPLIT_WARPS = (DRAIN_WARP0 - 2) / GROUPS;
  // registers per thread after reallocation, 64 K in all
  static constexpr int REGS_MOVERS = DRAIN_WARPS == 4 ? 96 : 72, REGS_DRAINERS = DRAIN_WARPS == 4 ? 216 : 184;
  static_assert(REGS_MOVERS * DRAIN_WARP0 * 32 + REGS_DRAINERS * DRAIN_WARPS * 32 <= 65536, "registers");
  static_assert(R >= L && TMEM_NEED <= 512 && SMEM <= 227 * 1024 - 512, "thin");
};

// First stage of share c of `cuts`.
__host__ __device__ inline int first_stage(int c, int cuts, int stages) {
  return static_cast<int>(static_cast<long long>(c) * stages / cuts);
}

template <int NT, int MP, bool A_KM>      // A_KM: the weights are [M, K]
__global__ void __launch_bounds__(THIN_THREADS, 1) thin_kernel(const __grid_constant__ ThinParams p) {
  using Cfg = ThinCfg<NT, MP, A_KM>;
  extern __shared__ uint8_t thin_smem[];
  __shared__ __align__(8) uint64_t bar_tma[8], bar_split[8], bar_empty[8], bar_tmem_full[2], bar_tmem_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t raw = (smem_u32(thin_smem) + 1023u) & ~1023u, lo = raw + Cfg::R * Cfg::RAW;
  constexpr uint32_t R = Cfg::R, L = Cfg::L;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < 8; ++i) {
      mbar_init(smem_u32(&bar_tma[i]), 1);
      mbar_init(smem_u32(&bar_split[i]), Cfg::SPLIT_WARPS);
      mbar_init(smem_u32(&bar_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_tmem_full[i]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[i]), Cfg::DRAIN_WARPS);
    }
    fence_mbar_init();
  }
  if (warp == 2) {
    tmem_alloc<1>(smem_u32(&tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int cuts = p.slices / p.items;
  // every role walks this block's slices: body(item, first stage, stage behind the last, slice)
  auto each_slice = [&](auto body) {
    for (int id = blockIdx.x; id < p.slices; id += gridDim.x) {
      const int c = id / p.items;
      if (!body(id - c * p.items, first_stage(c, cuts, p.stages), first_stage(c + 1, cuts, p.stages), id)) break;
    }
  };
  auto give_up = [&](int role, int a, int b) {
    abort_flag = 1;
    atomicCAS(p.status, 0, (role << 24) | ((a & 0xFF) << 16) | (b & 0xFFFF));
  };

  if (warp < Cfg::DRAIN_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_MOVERS));
    if (warp == 0) {
      // ---------------------------------------------------------- loads
      uint32_t s = 0, ph = 0, it = 0;
      uint32_t held = 0;                   // stages whose X has not been asked for yet
      int held_k[R];
      bool started = p.early == 0;
      auto load_x = [&](uint32_t slot, int k) {
        const CUtensorMap* map = k >= p.half ? &p.tmX[1] : &p.tmX[0];
        const int k0 = (k >= p.half ? k - p.half : k) * Cfg::KS * 32;
#pragma unroll
        for (int b = 0; b < Cfg::KS; ++b)
          tma_load_3d(raw + slot * Cfg::RAW + Cfg::W_BYTES + b * 2 * Cfg::X_BYTES, map, smem_u32(&bar_tma[slot]), k0 + b * 32, 0, 0,
                      0ull);
      };
      auto x_of_held = [&]() {             // weights may be asked for before X exists; X waits for the grid that writes it
        if (lane == 0) {
          asm volatile("griddepcontrol.wait;" ::: "memory");
          for (uint32_t i = 0; i < held; ++i) load_x(i, held_k[i]);
        }
        __syncwarp();
        started = true;
      };
      each_slice([&](int item, int k0, int k1, int) {
        for (int k = k0; k < k1; ++k, ++it) {
          if (!started && held == R) x_of_held();
          if (!mbar_wait(smem_u32(&bar_empty[s]), ph ^ 1u, &abort_flag)) {
            if (lane == 0) give_up(ROLE_THIN_LOAD, s, it);
            return false;
          }
          if (elect_one()) {
            const uint32_t bar = smem_u32(&bar_tma[s]), dst = raw + s * Cfg::RAW;
            mbar_arrive_expect_tx(bar, Cfg::W_BYTES + Cfg::KS * Cfg::X_BYTES);
            const bool other = MP == 1 && item >= p.blocks, later = k >= p.half;
            const int col = (other ? item - p.blocks : item) * 128, kk = later ? k - p.half : k;
#pragma unroll
            for (int b = 0; b < Cfg::SUBS; ++b) {
              const CUtensorMap* map = (MP == 2 ? b == 1 : other || later) ? &p.tmW[1] : &p.tmW[0];
              const int row = (MP == 2 ? kk : kk * Cfg::KS + b) * 32;
              if (A_KM) {
                tma_load_3d(dst + b * 16384, map, bar, row, col, 0, 0ull);
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) tma_load_3d(dst + b * 16384 + j * 4096, map, bar, col + j * 32, row, 0, 0ull);
              }
            }
            if (started) load_x(s, k);
          }
          __syncwarp();
          if (!started) held_k[held++] = k;
          if (++s == R) { s = 0; ph ^= 1u; }
        }
        return true;
      });
      if (!started) x_of_held();
      if (lane == 0 && abort_flag) {       // copies in flight land before shared memory is released
        for (uint32_t i = it > R ? it - R : 0u; i < it; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(smem_u32(&bar_tma[i % R]), (i / R) & 1u) && clock64() - t0 < 20000000LL) {
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- products
      constexpr uint32_t ID_WIDE = make_idesc_tf32(128, Cfg::CONCAT ? 2 * NT : NT, !A_KM, false);
      constexpr uint32_t ID_NT = make_idesc_tf32(128, NT, !A_KM, false);
      constexpr uint32_t A_LBO = A_KM ? 16u : 4096u, A_SBO = A_KM ? 1024u : 512u;
      constexpr uint32_t A_LT = A_KM ? SMEM_LAYOUT_SW128 : SMEM_LAYOUT_SW128_32B;
      constexpr uint64_t A_STEP = (A_KM ? 32 : 1024) >> 4, B_STEP = 32 >> 4;     // 8 rows of K
      uint32_t s = 0, ph = 0, l = 0, ch = 0;
      each_slice([&](int, int k0, int k1, int) {
        for (int k = k0, kk = 0; k < k1; ++k) {
          const bool first = kk == 0;
          const bool last = ++kk == p.chunk || k + 1 == k1;
          if (last) kk = 0;
          if (!mbar_wait(smem_u32(&bar_split[s]), ph, &abort_flag)) {
            if (lane == 0) give_up(ROLE_THIN_MMA, s, k);
            return false;
          }
          const uint32_t buf = ch & 1u;
          if (first && !mbar_wait(smem_u32(&bar_tmem_empty[buf]), ((ch >> 1) & 1u) ^ 1u, &abort_flag)) {
            if (lane == 0) give_up(ROLE_THIN_MMA, 50 + buf, k);
            return false;
          }
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int b = 0; b < Cfg::SUBS; ++b) {
              const uint32_t d = tmem + (buf * MP + (MP == 2 ? b : 0)) * Cfg::DCOLS;
              const uint32_t x = raw + s * Cfg::RAW + Cfg::W_BYTES + (MP == 2 ? 0 : b) * 2 * Cfg::X_BYTES;
              const uint64_t bx = make_smem_desc(x, 16u, 1024u, SMEM_LAYOUT_SW128);
              const uint64_t bxl = make_smem_desc(x + Cfg::X_BYTES, 16u, 1024u, SMEM_LAYOUT_SW128);
              const uint64_t a_hi = make_smem_desc(raw + s * Cfg::RAW + b * 16384, A_LBO, A_SBO, A_LT);
              const uint64_t a_lo = make_smem_desc(lo + l * Cfg::LO + b * 16384, A_LBO, A_SBO, A_LT);
              const uint32_t fresh = first && (MP == 2 || b == 0) ? 0u : 1u;
              if (Cfg::CONCAT) {
                // columns [0, NT): hi*hi; columns [NT, 2 NT): hi*lo, then lo*hi
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_tf32<1>(d, a_hi + j * A_STEP, bx + j * B_STEP, ID_WIDE, j == 0 ? fresh : 1u);
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_tf32<1>(d + NT, a_lo + j * A_STEP, bx + j * B_STEP, ID_NT, 1u);
              } else {
                // the small products first, while the truncating accumulator is small
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  umma_tf32<1>(d, a_lo + j * A_STEP, bx + j * B_STEP, ID_NT, j == 0 ? fresh : 1u);
                  umma_tf32<1>(d, a_hi + j * A_STEP, bxl + j * B_STEP, ID_NT, 1u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) umma_tf32<1>(d, a_hi + j * A_STEP, bx + j * B_STEP, ID_NT, 1u);
              }
            }
            umma_commit<1>(smem_u32(&bar_empty[s]));
            if (last) umma_commit<1>(smem_u32(&bar_tmem_full[buf]));
          }
          __syncwarp();
          if (++s == R) { s = 0; ph ^= 1u; }
          if (++l == L) l = 0;
          if (last) ++ch;
        }
        return true;
      });
    } else {
      // ---------------------------------------------------------- split
      const uint32_t group = (warp - 2) / Cfg::SPLIT_WARPS;
      const int st = ((warp - 2) % Cfg::SPLIT_WARPS) * 32 + lane;
      constexpr int NST = Cfg::SPLIT_WARPS * 32;
      constexpr int VW = Cfg::W_BYTES / 16, VX = Cfg::X_BYTES / 16;
      static_assert(VW % 32 == 0 && VX % 32 == 0, "a warp's 32 vectors are 512 contiguous bytes");
      uint32_t s = 0, ph = 0, l = 0, sp = 0, php = 0, it = 0;
      auto next_block = [&]() {
        if (++s == R) { s = 0; ph ^= 1u; }
        if (++l == L) l = 0;
        if (it + 1 > L && ++sp == R) { sp = 0; php ^= 1u; }      // (sp, php): stage it + 1 - L
        ++it;
      };
      each_slice([&](int, int k0, int k1, int) {
        for (int k = k0; k < k1; ++k, next_block()) {
          if (it % Cfg::GROUPS != group) continue;
          if (!mbar_wait(smem_u32(&bar_tma[s]), ph, &abort_flag)) {
            if (lane == 0) give_up(ROLE_THIN_SPLIT, s, it);
            return false;
          }
          if (L != R && it >= L) {           // the lo slot is free once the products of stage it - L are done
            if (!mbar_wait(smem_u32(&bar_empty[sp]), php, &abort_flag)) {
              if (lane == 0) give_up(ROLE_THIN_SPLIT, 100 + sp, it);
              return false;
            }
          }
          const uint32_t from = raw + s * Cfg::RAW, to_w = lo + l * Cfg::LO;
          auto lo_of = [](float4 x) {
            return make_float4(rn_tf32(x.x - trunc_tf32(x.x)), rn_tf32(x.y - trunc_tf32(x.y)), rn_tf32(x.z - trunc_tf32(x.z)),
                               rn_tf32(x.w - trunc_tf32(x.w)));
          };
          constexpr int PER = (VW + NST - 1) / NST, G = 4;
#pragma unroll
          for (int b = 0; b < PER; b += G) {
            float4 x[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
              const int v = st + (b + i) * NST;
              if (b + i < PER && v < VW) x[i] = lds2x64(from + (v - lane) * 16, lane);
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
              const int v = st + (b + i) * NST;
              if (b + i < PER && v < VW) sts2x64(to_w + (v - lane) * 16, lane, lo_of(x[i]));
            }
          }
#pragma unroll
          for (int b = 0; b < (Cfg::KS * VX + NST - 1) / NST; ++b) {
            const int v = st + b * NST, sub = v / VX;     // X of the sub-blocks, each with its lo part behind it
            if (v < Cfg::KS * VX) {
              const uint32_t at = from + Cfg::W_BYTES + sub * 2 * Cfg::X_BYTES + (v - sub * VX - lane) * 16;
              sts2x64(at + Cfg::X_BYTES, lane, lo_of(lds2x64(at, lane)));
            }
          }
          fence_proxy_async_smem();          // the tensor core reads these through the async proxy
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_split[s]));
        }
        return true;
      });
    }
  } else {
    // ------------------------------------------------------------ drain: tensor memory -> registers -> scratch
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::REGS_DRAINERS));
    constexpr int MINE = Cfg::MINE;
    const int q = warp & 3, m0 = MINE == MP ? 0 : (warp - Cfg::DRAIN_WARP0) >> 2;
    uint32_t ch = 0;
    each_slice([&](int, int k0, int k1, int id) {
      float acc[MINE][NT];
#pragma unroll
      for (int m = 0; m < MINE; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = 0.0f;
      for (int k = k0; k < k1; k += p.chunk, ++ch) {
        const uint32_t buf = ch & 1u;
        if (!mbar_wait(smem_u32(&bar_tmem_full[buf]), (ch >> 1) & 1u, &abort_flag)) {
          if (lane == 0) give_up(ROLE_THIN_DRAIN, buf, k);
          return false;
        }
        tc_fence_after();
#pragma unroll
        for (int m = 0; m < MINE; ++m) {
          const uint32_t at = tmem + (static_cast<uint32_t>(q * 32) << 16) + (buf * MP + m0 + m) * Cfg::DCOLS;
#pragma unroll
          for (int t = 0; t < NT; t += 16) {
            float big[16], small[16];
            tmem_ld_32x16(at + t, big);
            if (Cfg::CONCAT) tmem_ld_32x16(at + NT + t, small);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[m][t + j] += Cfg::CONCAT ? big[j] + small[j] : big[j];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_tmem_empty[buf]));
      }
      float* out = p.part + (static_cast<long long>(id) * MP + m0) * (NT * 128) + q * 32 + lane;
#pragma unroll
      for (int m = 0; m < MINE; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) out[(m * NT + t) * 128] = acc[m][t];
      return true;
    });
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
  }
}

// Matrices a gated slice takes.
constexpr int mats_per_slice(int rows) { return rows >= 64 ? 2 : 1; }

// Sums of a column block's slices in order, gate, rows out.  One 16-byte vector of a row per thread.
struct ThinSumParams {
  const float* part;
  float* out; float* G; float* U;
  const float* preG; const float* preU;      // gradients: the pre-activations; out, U = deltaG, deltaU
  int N, M, act, blocks, cuts;
};
template <int NT, int MATS, bool TOGETHER>      // TOGETHER: the slices held both matrices
__global__ void __launch_bounds__(256) thin_sum_kernel(const __grid_constant__ ThinSumParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int vecs = p.M / 4;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<long long>(p.N) * vecs;
       i += static_cast<long long>(gridDim.x) * 256) {
    const int n = static_cast<int>(i / vecs), v = static_cast<int>(i - static_cast<long long>(n) * vecs);
    const int block = v >> 5;
    float s[MATS * 4];
#pragma unroll
    for (int k = 0; k < MATS * 4; ++k) s[k] = 0.0f;
    auto part_of = [&](int c, int m, int blk) -> long long {
      return TOGETHER ? (static_cast<long long>(c) * p.blocks + blk) * 2 + m
                      : (static_cast<long long>(c) * MATS + m) * p.blocks + blk;
    };
    for (int b = 0; b < p.cuts; ++b) {
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        const float4 x = *reinterpret_cast<const float4*>(
            p.part + (part_of(b, m, block) * NT + n) * 128 + (v & 31) * 4);
        s[m * 4] += x.x; s[m * 4 + 1] += x.y; s[m * 4 + 2] += x.z; s[m * 4 + 3] += x.w;
      }
    }
    const long long at = static_cast<long long>(n) * p.M + v * 4;
    if constexpr (MATS == 2) {
      if (p.G != nullptr) {
        *reinterpret_cast<float4*>(p.G + at) = make_float4(s[0], s[1], s[2], s[3]);
        *reinterpret_cast<float4*>(p.U + at) = make_float4(s[4], s[5], s[6], s[7]);
      }
      gated_forward<4>(p.act, s);
    }
    if constexpr (MATS == 1) {
      if (p.preG != nullptr) {               // s is deltaH
        const float4 g = *reinterpret_cast<const float4*>(p.preG + at), u = *reinterpret_cast<const float4*>(p.preU + at);
        float4 dg, du;
        gated_backward4(p.act, make_float4(s[0], s[1], s[2], s[3]), g, u, &dg, &du);
        *reinterpret_cast<float4*>(p.out + at) = dg;
        *reinterpret_cast<float4*>(p.U + at) = du;
        continue;
      }
    }
    *reinterpret_cast<float4*>(p.out + at) = make_float4(s[0], s[1], s[2], s[3]);
  }
}

// Shares of K: the rounds of slices over the SMs times a slice's blocks of 32 rows (0.37 us of a block's way from memory
// each, five more for a slice's start and end), plus what the slices' sums cost to write and read again.
int cuts_of(int items, int kblocks, int rows, int mats) {
  const int sms = device_sm_count();
  int best = 1;
  double best_t = 1e300;
  for (int c = 1; c <= 32 && (c == 1 || kblocks / c >= 4); ++c) {
    const int rounds = (items * c + sms - 1) / sms;
    const double t = rounds * ((kblocks + c - 1) / c + 5) * mats * 0.37e-6 +
                     static_cast<double>(items) * c * mats * rows * 128 * 8 / 4e12;
    if (t < best_t) { best_t = t; best = c; }
  }
  return best;
}

// MATS matrices side by side, or (A_KM) the transposed ones, two of them summed.
template <int NT, int MATS, bool A_KM>
int thin_launch(const ThinCall& c, cudaStream_t st) {
  constexpr int MP = MATS == 2 ? mats_per_slice(NT) : 1;
  using Cfg = ThinCfg<NT, MP, A_KM>;
  auto kernel = thin_kernel<NT, MP, A_KM>;
  static std::atomic<int> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e != cudaSuccess) return static_cast<int>(e);
    ready[dev & 63].store(1, std::memory_order_release);
  }
  ThinParams p;
  std::memset(&p, 0, sizeof(p));
  const uint64_t n = c.N, k = c.K, m = c.M;
  auto weight_map = [&](CUtensorMap* map, const float* w) {
    return A_KM ? make_map3(map, w, k, m, 1, k, k * m, 32, 128, false) : make_map3(map, w, m, k, 1, m, m * k, 32, 32, true);
  };
  if (int rc = weight_map(&p.tmW[0], c.W0)) return rc;
  if (c.W1)
    if (int rc = weight_map(&p.tmW[1], c.W1)) return rc;
  if (int rc = make_map3(&p.tmX[0], c.X, k, n, 1, k, k * n, 32, NT, false)) return rc;
  if (c.X1)
    if (int rc = make_map3(&p.tmX[1], c.X1, k, n, 1, k, k * n, 32, NT, false)) return rc;
  p.part = c.work;
  const int kblocks = (c.K + 31) / 32;
  p.half = (kblocks + Cfg::KS - 1) / Cfg::KS;
  p.stages = c.X1 ? 2 * p.half : p.half;
  p.blocks = (c.M + 127) / 128;
  p.items = p.blocks * MATS / MP;
  const int cuts = cuts_of(p.items, c.X1 ? 2 * kblocks : kblocks, NT, MP);
  p.slices = p.items * cuts;
  p.chunk = (GATED_KC + Cfg::KS - 1) / Cfg::KS;
  p.early = c.early;
  p.status = status_word_ptr(&e);
  if (!p.status) return static_cast<int>(e);
  const int grid_x = p.slices < device_sm_count() ? p.slices : device_sm_count();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_x, 1, 1);
  cfg.blockDim = dim3(THIN_THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = c.early ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return static_cast<int>(e);
  ThinSumParams q{};
  q.part = c.work; q.out = c.out; q.G = c.G; q.U = c.U; q.preG = c.preG; q.preU = c.preU;
  q.N = c.N; q.M = c.M; q.act = c.act; q.blocks = p.blocks; q.cuts = cuts;
  const long long vecs = static_cast<long long>(c.N) * (c.M / 4);
  long long grid = (vecs + 255) / 256;
  if (grid > 8LL * device_sm_count()) grid = 8LL * device_sm_count();
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, thin_sum_kernel<NT, MATS, MP == 2>, q));
}

int thin_rows(int N) { return N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : 128; }

}  // namespace

long long thin_work_floats(int N, int M, int K, ThinForm form) {
  const int rows = thin_rows(N), mats = form == THIN_GATED ? 2 : 1, together = form == THIN_GATED ? mats_per_slice(rows) : 1;
  const int items = (M + 127) / 128 * mats / together, kblocks = (K + 31) / 32 * (form == THIN_DUAL ? 2 : 1);
  return static_cast<long long>(items) * cuts_of(items, kblocks, rows, together) * together * rows * 128;
}

int thin_product(const ThinCall& c, ThinForm form, cudaStream_t st) {
  if (!load_driver_entry_points()) return CU32_E_DRIVER;
  const int rows = thin_rows(c.N);
  switch (form) {
    case THIN_GATED:
      return rows == 16 ? thin_launch<16, 2, false>(c, st) : rows == 32 ? thin_launch<32, 2, false>(c, st)
             : rows == 64 ? thin_launch<64, 2, false>(c, st) : thin_launch<128, 2, false>(c, st);
    case THIN_PLAIN:
      return rows == 16 ? thin_launch<16, 1, false>(c, st) : rows == 32 ? thin_launch<32, 1, false>(c, st)
             : rows == 64 ? thin_launch<64, 1, false>(c, st) : thin_launch<128, 1, false>(c, st);
    default:
      return rows == 16 ? thin_launch<16, 1, true>(c, st) : rows == 32 ? thin_launch<32, 1, true>(c, st)
             : rows == 64 ? thin_launch<64, 1, true>(c, st) : thin_launch<128, 1, true>(c, st);
  }
}

}  // namespace dragon
