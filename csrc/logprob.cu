// Log-probabilities of given tokens under a linear head, and their gradient.
//
//   a[t, v]  = <h_t, w_v>                       tcgen05 product, fp32 accumulators
//   z[t, v]  = softcap(a) / temperature         softcap(a) = cap * tanh(a / cap), or a
//   out[t]   = z[t, y_t] - log sum_v exp z[t, v]
//   d out[t] / d a[t, v] = (onehot(y_t) - p[t, v]) * softcap'(a) / temperature,  p = softmax(z)
//
// The logits never reach memory: the product's epilogue turns each accumulator row of a
// tile into a running (reference, sum of 2^(z log2e - reference)) pair, and a second small
// kernel joins a row's pairs in a fixed order.
//
// Gradient. dh = G W and dW = G^T h with G[t, v] = g_t * d out[t] / d a[t, v], in bf16, but
// for the labels' entries, most of a gradient's norm: G has zeros there, and their part is
// added in fp32: one weight row to each row of dh (scatter_kernel), one hidden row for each
// token to dW (label_rows_kernel sums them, the product's epilogue adds them before its
// rounding). With them in G its rounding to bf16 would be as large as the output's (error of
// dW against 64 bits 0.0026, now the output's own 0.0017). The plain way recomputes each tile
// of the product in the backward pass (head_kernel STORE): 8 T V D operations in all. Large
// problems need 6: dh = diag(c) X W and dW = X^T diag(c) h hold for any X whose rows are G's
// up to factors c_t, so the forward pass already stores
//   X[t, v] = bf16(2^(z log2e - r_t) * softcap'(a)),   r_t = z[t, y_t] log2e + 40
// with a reference r_t that one dot product gives beforehand, and the backward pass folds c_t
// = -(g_t / temperature) 2^(r_t - lse2_t) into the hidden rows (for dW) and into the result
// (for dh). Both factors have to lie in bf16's range, 2^-126 to 2^127. X's entries reach at most
// 2^(-out log2e - 40), those of probability p are p times that, and c_t is g_t / temperature
// divided by it: kept up to 2^60 (out > -69 or so) the entries of p > 2^-86 and the c_t h_t of
// |g_t h_t| > 2^-66 are normal numbers. If any row is beyond that, a flag in device memory makes
// the backward pass recompute. What it costs: c_t h_t is rounded to bf16 (2^-8 of a term of dW
// other than the labels').
//
// Rows whose label is ignore_index are left out of the products: compact_kernel lists
// the others on the device, gather_kernel packs their hidden rows, and every later kernel reads
// the row count from device memory, so nothing is read back to the host and a NaN or an
// infinity in an ignored row reaches neither gradient.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "ops.h"

namespace plg {
namespace {

constexpr int kBM = 128;  // rows of a tile per CTA (256 per CTA pair)
constexpr int kBK = 64;   // one 128-byte swizzle row of bf16
constexpr int kMaxBN = 256;
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;  // a warpgroup of loads and MMAs, two of epilogue
// Registers of the warpgroups where the epilogue holds a whole accumulator row part: the
// launch has 168 for each of 384 threads, and 80 + 2 * 208 < 3 * 168.
constexpr int kLoadRegs = 80, kEpiRegs = 208;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kMaxStageBytes = kABytes + (kMaxBN / 2) * kBK * 2;
// per epilogue warp: two 32 x 32 bf16 boxes on their way to X
constexpr int kBoxBytes = 32 * 32 * 2;
constexpr int kSmemBytes = kStages * kMaxStageBytes + kEpiWarps * 2 * kBoxBytes + 1024 + 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRefOffset = 40.f;   // r_t - z_y log2e
constexpr float kRefLimit = 60.f;    // lse2 - r_t beyond which X is recomputed
// Reduction length of one accumulator of the statistics: the tensor cores truncate each
// addition, a bias of about 1e-9 of the sum per column of D (measured: 2.5e-6 of a logit at
// D = 2560, 1e-6 at 1024; an fp32 chain's rounding is about 5e-7), so longer sums are cut
// into pieces that the epilogue adds in fp32: of 1024 (512 cost 17% of the time at D = 1024;
// 1280 save 2% at D = 2560). Where the head's bytes bound the call, thin_kernel, pieces of 512
// are within 3% of those of 1024 (58.1 against 58.3 us for one row, D = 1024; relative error
// 5.8e-8 instead of 8.0e-8 rms, 3.9e-8 for fp32 throughout) and 256 cost 10%.
constexpr int kSegBlocks = 1024 / kBK, kThinSegBlocks = 512 / kBK;

struct HeadArgs {
  int rows, N, k_blocks, segs;
  int bn, n_tiles, group_m;
  const int* n_rows;            // device row count (null: rows)
  const int* row_map;           // compact row -> token (null: identity)
  const int64_t* labels;        // per token
  long long label0;             // vocabulary index of column 0
  float k;                      // log2(e) / temperature
  float cap, inv_cap;
  int* status;
  float2* part;                 // statistics: [rows][2 * n_tiles]
  float* target;                // statistics: [rows] a (after the softcap) of the label
  const float* ref;             // X: [rows] r_t
  const float* gout;            // X alone: per token
  float inv_temp;
  const int* only_if;           // X alone: nothing to do unless this device flag is set
};

__device__ __forceinline__ float ex2(float x) { return fast_exp2(x); }

// y = v where lane index `at` is i: a predicated move, which keeps a register array that is
// searched for one element from becoming an indexed array in local memory
__device__ __forceinline__ void pick_if(float& y, float v, int at, int i) {
  asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %2, %3;\n\t@p mov.f32 %0, %1;\n\t}"
      : "+f"(y)
      : "f"(v), "r"(at), "r"(i));
}

// Persistent CTA-pair kernel: 256 x bn tiles with tcgen05.mma.cta_group::2. CTA rank r
// holds rows [128 r, 128 r + 128) of the tile and loads those of A and half of B's bn
// columns. Warp 0 loads (TMA), warp 1 of rank 0 issues the MMAs, warps 4 to 11 drain the
// accumulator (two warps per 32-row quadrant, alternate 32-column chunks), double
// buffered in TMEM against the next main loop. STATS: the rows' (reference, sum) pairs;
// STORE: X, staged per warp and written by TMA; SEG: more than one accumulator piece.
// 256 x 256 tiles because two CTAs that share B halve its loads: 64 KB of operands for 2^22
// multiply-adds of a pair, below what L2 gives. Bound by the tensor cores, and in long runs by
// the power they draw: statistics alone of 4096 x 151936, D = 2560: 2.12 ms, 1500 TFLOP/s (0.89
// of the measured burst rate); with X of 5308 x 128256, D = 2048, in a long run at 1320 MHz 2.42
// ms, 1150 TFLOP/s, where the library's product alone, its bf16 logits written, takes 2.17. The
// epilogue hides behind the next main loop (tensor pipe 73% busy at 4096 x 32768, D = 1024, X
// written).
template <bool STATS, bool STORE, bool CAP, bool SEG>
__global__ void __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmX, const HeadArgs args) {
  if (!STATS && args.only_if != nullptr && *args.only_if == 0) return;  // uniform over the grid
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* boxes = smem + kStages * kMaxStageBytes;
  uint64_t* bar = reinterpret_cast<uint64_t*>(boxes + kEpiWarps * 2 * kBoxBytes);
  uint64_t* full_bar = bar;                  // [kStages] (rank 0's are used)
  uint64_t* empty_bar = bar + kStages;       // [kStages]
  uint64_t* accf_bar = bar + 2 * kStages;    // [2]
  uint64_t* acce_bar = bar + 2 * kStages + 2;  // [2] (rank 0's are used)
  uint64_t* done_bar = bar + 2 * kStages + 4;
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bar + 2 * kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_smem + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int bn = args.bn;
  const uint32_t stage_bytes = kABytes + (bn / 2) * kBK * 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 2 * kEpiWarps);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (STORE) tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_base_smem, 512);
    tmem_relinquish_pair();
  }
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_smem;

  // rows in use: every role of both CTAs reads the same device count
  const int rows = args.n_rows != nullptr ? min(*args.n_rows, args.rows) : args.rows;
  const int m_tiles = (rows + 2 * kBM - 1) / (2 * kBM);
  const int total = m_tiles * args.n_tiles;
  const int segs = SEG ? args.segs : 1;
  // m tiles walk fastest within a group of group_m of them, so the group's rows stay in L2
  // while the head streams past once per group
  auto decode = [&](int w, int& mt, int& nt) {
    const int per_group = args.group_m * args.n_tiles;
    const int g = w / per_group;
    const int m0 = g * args.group_m;
    const int gm = min(args.group_m, m_tiles - m0);
    const int r = w - g * per_group;
    nt = r / gm;
    mt = m0 + (r - nt * gm);
  };

  if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    if (SEG) setmaxnreg_inc<kEpiRegs>();  // heads its warpgroups' branch
    const int q = warp & 3;           // TMEM lane quadrant this warp may access
    const int half = (warp - 4) >> 2;  // which of the quadrant's two warps
    const int chunks = bn / 32;
    uint8_t* box = boxes + (warp - 4) * 2 * kBoxBytes;
    int local = 0, nbox = 0;
    bool ok = true;
    for (int w = pair; w < total && ok; w += npairs) {
      int mt, nt;
      decode(w, mt, nt);
      const int row0 = mt * 2 * kBM + static_cast<int>(rank) * kBM + q * 32;  // the warp's first row
      const int row = row0 + lane;
      const bool live = row < rows;
      // this row's label as a column of this launch, and its constants
      long long lab = -1;
      float rref = 0.f, coef = 0.f;
      if (live) {
        const int tok = args.row_map != nullptr ? args.row_map[row] : row;
        lab = args.labels[tok] - args.label0;
        if (STORE) rref = args.ref[row];
        if (STORE && !STATS) coef = args.gout[tok] * args.inv_temp;
      }
      // warps without any row in use skip the math (X gets its zero rows all the same)
      const bool busy = STORE ? row0 < args.rows : row0 < rows;
      float acc[SEG ? 4 : 1][32];
      for (int seg = 0; seg < segs; ++seg, ++local) {
        const int buf = local & 1;
        if (!mbar_wait_bounded(&accf_bar[buf], (local >> 1) & 1, abort_flag)) {
          record_status(args.status, kTimeoutAccFull);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * kMaxBN;
        if (SEG && busy) {
#pragma unroll
          for (int j = 0; j < (SEG ? 4 : 1); ++j) {
            if (half + 2 * j >= chunks) continue;
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              uint32_t r[16];
              __syncwarp();
              tmem_ld_32x32b_x16(t_row + (half + 2 * j) * 32 + h, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                acc[j][h + i] = __uint_as_float(r[i]) + (seg == 0 ? 0.f : acc[j][h + i]);
            }
          }
        }
        if (SEG) {  // the row part is in registers: the next main loop may have the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(&acce_bar[buf], 0);
        }
        if (busy && seg == segs - 1) {
          float ref = -INFINITY, s0 = 0.f, s1 = 0.f, target = 0.f;
          auto chunk = [&](int c, float (&v)[32]) __attribute__((always_inline)) {
            const int col0 = nt * bn + c * 32;
            if (col0 >= args.N) return;  // uniform over the warp
            float slope[CAP && STORE ? 32 : 1];
            if (CAP) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float t = tanhf(v[i] * args.inv_cap);
                v[i] = args.cap * t;
                if (STORE) slope[i] = 1.f - t * t;
              }
            }
            const int lc = (lab >= col0 && lab < col0 + 32) ? static_cast<int>(lab - col0) : -1;
            if (STATS) {
              // With whole row parts in registers the pick runs unconditionally: a branch around
              // it makes the compiler spill 80 registers, and the long main loop hides it.
              if (SEG || __any_sync(0xffffffffu, lc >= 0)) {
#pragma unroll
                for (int i = 0; i < 32; ++i) pick_if(target, v[i], lc, i);
              }
              if (col0 + 32 > args.N) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (col0 + i >= args.N) v[i] = -INFINITY;
              }
              float m = fmax3(v[0], v[1], v[2]);
#pragma unroll
              for (int i = 3; i < 31; i += 2) m = fmax3(m, v[i], v[i + 1]);
              m = fmaxf(m, v[31]);
              const float nref = fmaxf(ref, m * args.k);
              const float sub = nref == -INFINITY ? 0.f : nref;
              const float f = ex2(ref - sub);
              s0 *= f;
              s1 *= f;
              ref = nref;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float e0, e1;
                ffma2(e0, e1, v[i], v[i + 1], args.k, args.k, -sub, -sub);
                v[i] = ex2(e0);
                v[i + 1] = ex2(e1);
                fadd2(s0, s1, s0, s1, v[i], v[i + 1]);
              }
              if (STORE) {
                const float to_ref = nref == -INFINITY ? 0.f : ex2(sub - rref);
#pragma unroll
                for (int i = 0; i < 32; i += 2) fmul2(v[i], v[i + 1], v[i], v[i + 1], to_ref, to_ref);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float e0, e1;
                ffma2(e0, e1, v[i], v[i + 1], args.k, args.k, -rref, -rref);
                v[i] = ex2(e0);
                v[i + 1] = ex2(e1);
              }
            }
            if (STORE) {
              uint32_t o[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                if (CAP) {
                  v[i] *= slope[i % (CAP && STORE ? 32 : 1)];
                  v[i + 1] *= slope[(i + 1) % (CAP && STORE ? 32 : 1)];
                }
                if (!STATS) {
                  v[i] = i == lc ? 0.f : -coef * v[i];
                  v[i + 1] = i + 1 == lc ? 0.f : -coef * v[i + 1];
                }
                // rows past the count up to the tile's end: zero padding of the products
                o[i / 2] = live ? pack_bf16x2(v[i], v[i + 1]) : 0u;
              }
              // 64-byte rows, 16-byte pieces swizzled as the tensor map expects them
              uint8_t* b = box + (nbox & 1) * kBoxBytes;
              if (lane == 0) bulk_wait_group_read<1>();
              __syncwarp();
              uint4* brow = reinterpret_cast<uint4*>(b + lane * 64);
#pragma unroll
              for (int p = 0; p < 4; ++p)
                brow[p ^ ((lane >> 1) & 3)] = make_uint4(o[4 * p], o[4 * p + 1], o[4 * p + 2], o[4 * p + 3]);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&tmX, b, col0, row0);
                bulk_commit_group();
              }
              ++nbox;
            }
          };
          if (SEG) {
#pragma unroll
            for (int j = 0; j < (SEG ? 4 : 1); ++j)
              if (half + 2 * j < chunks) chunk(half + 2 * j, acc[j]);
          } else {
#pragma unroll 1
            for (int c = half; c < chunks; c += 2) {
              uint32_t r[32];
              __syncwarp();
              tmem_ld_32x32b_x32(t_row + c * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) acc[0][i] = __uint_as_float(r[i]);
              chunk(c, acc[0]);
            }
          }
          // the label's chunk was one of this warp's
          if (STATS && lab >= nt * bn && lab < min((nt + 1) * bn, args.N) &&
              ((static_cast<int>(lab) - nt * bn) / 32) % 2 == half)
            args.target[row] = target;
          if (STATS && live)
            args.part[static_cast<long long>(row) * (2 * args.n_tiles) + 2 * nt + half] =
                make_float2(ref, s0 + s1);
        }
        if (!SEG) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(&acce_bar[buf], 0);
        }
      }
    }
    // the staged boxes must have left shared memory (and reached X) before the CTA exits
    if (STORE && lane == 0) bulk_wait_group<0>();
  } else {
    if (SEG) setmaxnreg_dec<kLoadRegs>();
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        uint32_t armed_mask = 0, parity_mask = 0;
        for (int w = pair; w < total && ok; w += npairs) {
          int mt, nt;
          decode(w, mt, nt);
          const int m0 = mt * 2 * kBM + static_cast<int>(rank) * kBM;
          const int n0 = nt * bn + static_cast<int>(rank) * (bn / 2);
          for (int kb = 0; kb < args.k_blocks; ++kb) {
            if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag)) {
              record_status(args.status, kTimeoutSmemEmpty);
              *abort_flag = 1;
              ok = false;
              break;
            }
            uint8_t* sA = smem + stage * kMaxStageBytes;
            if (leader) {
              mbar_arrive_expect_tx(&full_bar[stage], 2 * stage_bytes);
              armed_mask |= 1u << stage;
              parity_mask = (parity_mask & ~(1u << stage)) | (phase << stage);
            }
            tma_load_2d_pair(sA, &tmA, &full_bar[stage], kb * kBK, m0);
            tma_load_2d_pair(sA + kABytes, &tmB, &full_bar[stage], kb * kBK, n0);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        if (!ok) {
          // unwind: let the copies in flight land before the CTA can exit
          if (leader) {
            for (int s = 0; s < kStages; ++s)
              if (((armed_mask >> s) & 1u) &&
                  !mbar_wait_bounded(&full_bar[s], (parity_mask >> s) & 1u, nullptr))
                record_status(args.status, kTimeoutDrain);
          } else {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 2000000ull) {
            }
          }
        }
      }
    } else if (warp == 1) {
      // ----------------------------------------------------------------- MMA
      if (lane == 0 && leader) {
        const uint32_t idesc = make_idesc_bf16_f32(2 * kBM, bn, false, false);
        int stage = 0;
        uint32_t phase = 0;
        int local = 0;
        bool ok = true;
        for (int w = pair; w < total && ok; w += npairs) {
          for (int seg = 0; seg < segs && ok; ++seg, ++local) {
            const int kb0 = seg * args.k_blocks / segs, kb1 = (seg + 1) * args.k_blocks / segs;
            const int buf = local & 1;
            const uint32_t acc_phase = (local >> 1) & 1;
            if (!mbar_wait_bounded(&acce_bar[buf], acc_phase ^ 1u, abort_flag)) {
              record_status(args.status, kTimeoutAccEmpty);
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + buf * kMaxBN;
            for (int kb = kb0; kb < kb1; ++kb) {
              if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag)) {
                record_status(args.status, kTimeoutTmaFull);
                *abort_flag = 1;
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t sA = smem_u32(smem + stage * kMaxStageBytes);
              const uint64_t da0 = make_smem_desc(sA, 16, 1024, kLayoutSW128);
              const uint64_t db0 = make_smem_desc(sA + kABytes, 16, 1024, kLayoutSW128);
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk)
                tc_mma_ss_pair(d_tmem, desc_advance(da0, kk * 32), desc_advance(db0, kk * 32), idesc,
                               (kb > kb0 || kk > 0) ? 1u : 0u);
              tc_commit_pair(&empty_bar[stage], 0x3);
              if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
              }
            }
            if (ok) tc_commit_pair(&accf_bar[buf], 0x3);
          }
        }
        if (!ok) *abort_flag = 1;
        tc_commit_pair(done_bar, 0x3);
      }
      if (lane == 0 && !mbar_wait_bounded(done_bar, 0, nullptr)) record_status(args.status, kTimeoutDrain);
      __syncwarp();
    }
  }

  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- few rows
// Scoring at most 128 rows is one pass through the head, bound by its bytes. Here the roles
// are swapped: 128 vocabulary entries are the tensor core's rows and the NT (32, 64 or 128)
// hidden rows its columns, so that an MMA costs in proportion to the rows in use. CTA c takes
// the entries [V c / CTAs, V (c + 1) / CTAs), equal shares of the bytes for every SM, in
// equal tiles of at most 128 entries (the other kernel's 594 tiles of 256 columns are 9 waves
// over 74 SM pairs for 8.03 waves of work).
// Accumulator lane = entry, column = hidden row: a warp reduces 32 entries x 32 rows by
// exchanging halves (31 shuffles instead of 160), which leaves lane j with row j's result,
// and keeps each row's running (reference, sum) there. One pair per row, CTA and quadrant.
// One row, D = 1024, V = 151936 (311 MB): 55 us, 5.7 TB/s; the call 57 us.
// 128 rows: the call 66 us (129, by the other kernel: 83). D = 2560: 6.2 TB/s, 0.95 of the measured copy rate.
constexpr int kThinThreads = 192;
constexpr int kThinEntries = 128;

template <int NT>
struct Thin {
  static constexpr int kA = kThinEntries * kBK * 2;
  static constexpr int kB = NT * kBK * 2;
  static constexpr int kStages = NT == 128 ? 6 : (NT == 64 ? 8 : 10);
  static constexpr int kSmem = kStages * (kA + kB) + 1024 + 256;
};

struct ThinArgs {
  int T, V, tile, k_blocks, segs;
  const int64_t* labels;
  float k, cap, inv_cap;
  float2* part;   // [T][4 * CTAs]
  float* target;  // [T]
  int* status;
};

// lane j of the result = op over the lanes of column j: each step keeps one half of the
// columns and trades the other half with the lane whose index differs in that bit
template <typename Op>
__device__ __forceinline__ float transpose_reduce(const float (&v)[32], int lane, Op op) {
  float t[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const bool hi = lane & 16;
    const float send = hi ? v[i] : v[i + 16], keep = hi ? v[i + 16] : v[i];
    t[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, 16));
  }
#pragma unroll
  for (int w = 8; w >= 1; w >>= 1) {
    const bool hi = lane & w;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float send = hi ? t[i] : t[i + w], keep = hi ? t[i + w] : t[i];
      t[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, w));
    }
  }
  return t[0];
}

template <int NT, bool CAP>
__global__ void __launch_bounds__(kThinThreads, 1)
    thin_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmH,
                const ThinArgs args) {
  using C_ = Thin<NT>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C_::kStages * (C_::kA + C_::kB));
  uint64_t* full_bar = bar;
  uint64_t* empty_bar = bar + C_::kStages;
  uint64_t* accf_bar = bar + 2 * C_::kStages;      // [2]
  uint64_t* acce_bar = bar + 2 * C_::kStages + 2;  // [2]
  uint64_t* done_bar = bar + 2 * C_::kStages + 4;
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(bar + 2 * C_::kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_smem + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  dependents_may_start();

  if (threadIdx.x == 0) {
    for (int s = 0; s < C_::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf_bar[b], 1);
      mbar_init(&acce_bar[b], 4);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_smem, 2 * NT);
    tmem_relinquish();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_smem;
  const int v0 = static_cast<int>(static_cast<long long>(args.V) * blockIdx.x / gridDim.x);
  const int v1 = static_cast<int>(static_cast<long long>(args.V) * (blockIdx.x + 1) / gridDim.x);
  const int tiles = (v1 - v0 + args.tile - 1) / args.tile;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool ok = true;
      const uint32_t bytes = args.tile * kBK * 2 + C_::kB;
      for (int i = 0; i < tiles && ok; ++i) {
        for (int kb = 0; kb < args.k_blocks; ++kb) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            record_status(args.status, kTimeoutSmemEmpty);
            *abort_flag = 1;
            ok = false;
            break;
          }
          uint8_t* sA = smem + stage * (C_::kA + C_::kB);
          mbar_arrive_expect_tx(&full_bar[stage], bytes);
          tma_load_2d(sA, &tmW, &full_bar[stage], kb * kBK, v0 + i * args.tile);
          tma_load_2d(sA + C_::kA, &tmH, &full_bar[stage], kb * kBK, 0);
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == C_::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        for (int s = 0; s < C_::kStages; ++s)
          if (((issued >> s) & 1u) && !mbar_wait_bounded(&full_bar[s], (parity >> s) & 1u, nullptr))
            record_status(args.status, kTimeoutDrain);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- MMA
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_bf16_f32(kThinEntries, NT, false, false);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        for (int seg = 0; seg < args.segs && ok; ++seg, ++local) {
          const int kb0 = seg * args.k_blocks / args.segs, kb1 = (seg + 1) * args.k_blocks / args.segs;
          const int buf = local & 1;
          if (!mbar_wait_bounded(&acce_bar[buf], ((local >> 1) & 1) ^ 1u, abort_flag)) {
            record_status(args.status, kTimeoutAccEmpty);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_bounded(&full_bar[stage], phase, abort_flag)) {
              record_status(args.status, kTimeoutTmaFull);
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sA = smem_u32(smem + stage * (C_::kA + C_::kB));
            const uint64_t da = make_smem_desc(sA, 16, 1024, kLayoutSW128);
            const uint64_t db = make_smem_desc(sA + C_::kA, 16, 1024, kLayoutSW128);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              tc_mma_ss(tmem_base + buf * NT, desc_advance(da, kk * 32), desc_advance(db, kk * 32), idesc,
                        (kb > kb0 || kk > 0) ? 1u : 0u);
            tc_commit(&empty_bar[stage]);
            if (++stage == C_::kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) tc_commit(&accf_bar[buf]);
        }
      }
      tc_commit(done_bar);
      if (!mbar_wait_bounded(done_bar, 0, nullptr)) record_status(args.status, kTimeoutDrain);
    }
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int kCh = NT / 32;
    const int q = warp & 3;
    float ref[kCh], sum[kCh];
    int lab[kCh];  // the label of hidden row 32 c + lane (never in a tile if there is none)
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      ref[c] = -INFINITY;
      sum[c] = 0.f;
      lab[c] = -1;
      if (c * 32 + lane < args.T) {
        const int64_t y = args.labels[c * 32 + lane];
        lab[c] = y >= 0 && y < args.V ? static_cast<int>(y) : -1;
      }
    }
    int local = 0;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int e0 = v0 + i * args.tile + q * 32;              // the warp's first entry
      const int end = min(v1, v0 + (i + 1) * args.tile);       // of the tile
      float acc[kCh][32];
      for (int seg = 0; seg < args.segs; ++seg, ++local) {
        const int buf = local & 1;
        if (!mbar_wait_bounded(&accf_bar[buf], (local >> 1) & 1, abort_flag)) {
          record_status(args.status, kTimeoutAccFull);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          uint32_t r[32];
          __syncwarp();
          tmem_ld_32x32b_x32(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * NT + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c][j] = __uint_as_float(r[j]) + (seg == 0 ? 0.f : acc[c][j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acce_bar[buf]);
      }
      if (!ok || e0 >= end) continue;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        if (c * 32 >= args.T) continue;
        float(&v)[32] = acc[c];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (CAP) v[j] = args.cap * tanhf(v[j] * args.inv_cap);
          if (e0 + lane >= end) v[j] = -INFINITY;
        }
        if (__any_sync(0xffffffffu, lab[c] >= e0 && lab[c] < min(e0 + 32, end))) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (__shfl_sync(0xffffffffu, lab[c], j) == e0 + lane && e0 + lane < end)
              args.target[c * 32 + j] = v[j];
        }
        const float m = transpose_reduce(v, lane, [](float a, float b) { return fmaxf(a, b); });
        const float nref = fmaxf(ref[c], m * args.k);
        const float sub = nref == -INFINITY ? 0.f : nref;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = ex2(fmaf(v[j], args.k, -__shfl_sync(0xffffffffu, sub, j)));
        const float s = transpose_reduce(v, lane, [](float a, float b) { return a + b; });
        sum[c] = sum[c] * ex2(ref[c] - sub) + s;
        ref[c] = nref;
      }
    }
#pragma unroll
    for (int c = 0; c < kCh; ++c)
      if (c * 32 + lane < args.T)
        args.part[(c * 32 + lane) * (4LL * gridDim.x) + 4 * blockIdx.x + q] = make_float2(ref[c], sum[c]);
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * NT);
  }
}

// ---------------------------------------------------------------- small kernels
constexpr int kScan = 1024;

// Block b lists the kept tokens of [1024 b, 1024 b + 1024): row_map (compact -> token, in
// token order), inverse (token -> compact or -1); ignored tokens get out = 0, labels
// outside the vocabulary NaN (and no gradient). The block counts the kept tokens before
// its own range itself, so one launch does the scan; the last block writes the total. Bound by
// latency (8192 tokens: 5 us, 0.4% of the products that follow).
__global__ void __launch_bounds__(kScan) compact_kernel(const int64_t* __restrict__ labels, long long T,
                                                        long long V, long long ignore_index,
                                                        int* __restrict__ row_map,
                                                        int* __restrict__ inverse,
                                                        int* __restrict__ count,
                                                        float* __restrict__ out) {
  __shared__ int s_warp[32];
  __shared__ int s_base;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    count[1] = 0;  // the flag that join_kernel may set
    count[2] = 1;  // k splits of dh's product, which may choose more
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long b0 = static_cast<long long>(blockIdx.x) * kScan;
  int before = 0;
  for (long long t = threadIdx.x; t < b0; t += kScan) {
    const int64_t y = labels[t];
    before += (y != ignore_index && y >= 0 && y < V) ? 1 : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) s_warp[warp] = before;
  __syncthreads();
  if (warp == 0) {
    int v = s_warp[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) s_base = v;
  }
  __syncthreads();
  const int base = s_base;
  const long long t = b0 + threadIdx.x;
  bool keep = false, bad = false;
  if (t < T) {
    const int64_t y = labels[t];
    bad = y != ignore_index && (y < 0 || y >= V);
    keep = y != ignore_index && !bad;
  }
  const unsigned bits = __ballot_sync(0xffffffffu, keep);
  if (lane == 0) s_warp[warp] = __popc(bits);
  __syncthreads();
  int off = base;
  for (int i = 0; i < warp; ++i) off += s_warp[i];
  off += __popc(bits & ((1u << lane) - 1u));
  if (t < T) {
    inverse[t] = keep ? off : -1;
    if (keep) row_map[off] = static_cast<int>(t);
    else out[t] = bad ? __int_as_float(0x7fc00000) : 0.f;
  }
  if (t == T - 1) *count = off + (keep ? 1 : 0);
}

// Packed bf16 hidden rows of the kept tokens; zero rows up to the next multiple of 256.
// With ref, also r_t = softcap(<h_t, w_{y_t}>) log2(e) / temperature + 40 of each row. Bound by
// memory, the label's weight row included (16384 rows, D = 1024: 33 us, 3 TB/s).
template <typename T>
__global__ void __launch_bounds__(128) gather_kernel(const T* __restrict__ h, long long ldh, int D,
                                                     const int* __restrict__ row_map,
                                                     const int* __restrict__ count,
                                                     __nv_bfloat16* __restrict__ out, int cap_rows,
                                                     const __nv_bfloat16* __restrict__ w, long long ldw,
                                                     const int64_t* __restrict__ labels, float k, float cap,
                                                     float* __restrict__ ref) {
  __shared__ float s_dot[2][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = *count;
  const int pad = min(cap_rows, (n + 255) / 256 * 256);
  int flip = 0;
  for (int r = blockIdx.x; r < pad; r += gridDim.x) {
    uint4* dst = reinterpret_cast<uint4*>(out + static_cast<long long>(r) * D);
    if (r >= n) {
      for (int i = threadIdx.x; i < D / 8; i += blockDim.x) dst[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const int tok = row_map[r];
    const T* src = h + static_cast<long long>(tok) * ldh;
    const uint4* wr = ref != nullptr ? reinterpret_cast<const uint4*>(w + labels[tok] * ldw) : nullptr;
    float dot = 0.f;
    for (int i = threadIdx.x; i < D / 8; i += blockDim.x) {
      uint4 u;
      if (sizeof(T) == 2) {
        u = reinterpret_cast<const uint4*>(src)[i];
      } else {
        const float4 a = reinterpret_cast<const float4*>(src)[2 * i];
        const float4 b = reinterpret_cast<const float4*>(src)[2 * i + 1];
        u = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                       pack_bf16x2(b.z, b.w));
      }
      dst[i] = u;
      if (ref != nullptr) {
        const uint4 v = wr[i];
        const uint32_t* up = &u.x;
        const uint32_t* vp = &v.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 a = unpack_bf16x2(up[j]), b = unpack_bf16x2(vp[j]);
          dot = fmaf(a.x, b.x, fmaf(a.y, b.y, dot));
        }
      }
    }
    if (ref != nullptr) {
      dot = warp_sum(dot);
      if (lane == 0) s_dot[flip][warp] = dot;
      __syncthreads();
      if (threadIdx.x == 0) {
        float a = s_dot[flip][0] + s_dot[flip][1] + s_dot[flip][2] + s_dot[flip][3];
        if (cap > 0.f) a = cap * tanhf(a / cap);
        ref[r] = fmaf(a, k, kRefOffset);
      }
      flip ^= 1;  // the next row's partial sums go to the other slots
    }
  }
}

// Joins a row's (reference, sum) pairs (thread-strided, then fixed shuffle trees: the same
// order every run) and writes out = z_label - lse. WARPS warps take a row: one where rows
// are many, a block of 8 where a few rows' pairs are all there is to read. Bound by memory
// (16384 rows of 1188 pairs, 156 MB: 40 us, 3.9 TB/s).
// For the gradient: lse2, (1 - p_y) softcap'(a_y), and the flag when X leaves bf16's range.
template <int WARPS>
__global__ void __launch_bounds__(256) join_kernel(const float2* __restrict__ part, int parts, int rows_,
                                                   const int* __restrict__ n_rows,
                                                   const int* __restrict__ row_map,
                                                   const int64_t* __restrict__ labels, long long V,
                                                   long long ignore_index,
                                                   const float* __restrict__ target, float k, float cap,
                                                   float* __restrict__ out, const float* __restrict__ ref,
                                                   float* __restrict__ lse2, float* __restrict__ label_grad,
                                                   int* __restrict__ flag) {
  __shared__ float2 s_part[8];
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kRows = 8 / WARPS;  // rows of a block
  const int sub = WARPS == 1 ? lane : threadIdx.x;
  const int rows = n_rows != nullptr ? min(*n_rows, rows_) : rows_;
  for (int r0 = blockIdx.x * kRows; r0 < rows; r0 += gridDim.x * kRows) {
    const int row = r0 + (WARPS == 1 ? warp : 0);
    float m = -INFINITY, s = 0.f;
    if (row < rows) {
      const float2* p = part + static_cast<long long>(row) * parts;
#pragma unroll 4
      for (int i = sub; i < parts; i += 32 * WARPS) {
        const float2 v = p[i];
        const float nm = fmaxf(m, v.x), off = nm == -INFINITY ? 0.f : nm;
        s = s * ex2(m - off) + v.y * ex2(v.x - off);
        m = nm;
      }
    }
    auto join = [&](float om, float os) {
      const float nm = fmaxf(m, om), off = nm == -INFINITY ? 0.f : nm;
      s = s * ex2(m - off) + os * ex2(om - off);
      m = nm;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o);
      const float os = __shfl_xor_sync(0xffffffffu, s, o);
      join(om, os);
    }
    if (WARPS > 1) {
      __syncthreads();
      if (lane == 0) s_part[warp] = make_float2(m, s);
      __syncthreads();
      m = s_part[0].x;
      s = s_part[0].y;
#pragma unroll
      for (int i = 1; i < WARPS; ++i) join(s_part[i].x, s_part[i].y);
    }
    if (row < rows && sub == 0) {
      const int tok = row_map != nullptr ? row_map[row] : row;
      const int64_t y = labels[tok];
      const float l2 = log2f(s);
      float v = 0.f;
      if (y != ignore_index)
        v = (y >= 0 && y < V) ? kLn2 * (fmaf(target[row], k, -m) - l2) : __int_as_float(0x7fc00000);
      out[tok] = v;
      if (lse2 != nullptr) {
        const float t = cap > 0.f ? target[row] / cap : 0.f;
        lse2[row] = m + l2;
        label_grad[row] = -expm1f(v) * (1.f - t * t);
        if (ref != nullptr && !(m + l2 - ref[row] <= kRefLimit)) *flag = 1;
      }
    }
  }
}

// Completes a kept X. Per row: c_t, the bf16 row c_t h_t, and a 0 at the label. Under the flag X
// has been recomputed as the gradient rows themselves: c_t = 1. Bound by memory (16384 rows, D =
// 1024: 19 us, 3.4 TB/s).
__global__ void __launch_bounds__(128) scale_rows_kernel(const __nv_bfloat16* __restrict__ h, int D,
                                                         const int* __restrict__ row_map,
                                                         const int* __restrict__ count,
                                                         const int64_t* __restrict__ labels,
                                                         const float* __restrict__ lse2,
                                                         const float* __restrict__ ref,
                                                         const float* __restrict__ gout, float inv_temp,
                                                         __nv_bfloat16* __restrict__ X, long long ldx,
                                                         float* __restrict__ scale,
                                                         __nv_bfloat16* __restrict__ hs, int cap_rows) {
  const int n = count[0];
  const bool whole = count[1] != 0;
  const int pad = min(cap_rows, (n + 255) / 256 * 256);
  for (int r = blockIdx.x; r < pad; r += gridDim.x) {
    uint4* dst = reinterpret_cast<uint4*>(hs + static_cast<long long>(r) * D);
    if (r >= n) {
      for (int i = threadIdx.x; i < D / 8; i += blockDim.x) dst[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const int tok = row_map[r];
    float c = 1.f;
    if (!whole) {
      c = -gout[tok] * inv_temp * exp2f(ref[r] - lse2[r]);
      if (threadIdx.x == 0) X[r * ldx + labels[tok]] = __float2bfloat16(0.f);
    }
    if (threadIdx.x == 0) scale[r] = c;
    const uint4* src = reinterpret_cast<const uint4*>(h + static_cast<long long>(r) * D);
    for (int i = threadIdx.x; i < D / 8; i += blockDim.x) {
      uint4 u = src[i];
      uint32_t* up = &u.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = unpack_bf16x2(up[j]);
        up[j] = pack_bf16x2(a.x * c, a.y * c);
      }
      dst[i] = u;
    }
  }
}

// dh[token] in dh's type from the compact fp32 rows (the sum of the product's k splits, in
// their order; times c_t with a kept X) plus the label's part, its entry of G times its weight
// row; zeros for the tokens left out. Bound by memory (16384 x 1024, two splits: 64 us, 3.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) scatter_kernel(const float* __restrict__ src, long long split_stride,
                                                      const int* __restrict__ splits,
                                                      const float* __restrict__ scale,
                                                      const float* __restrict__ label_grad,
                                                      const float* __restrict__ gout, float inv_temp,
                                                      const __nv_bfloat16* __restrict__ w, long long ldw,
                                                      const int64_t* __restrict__ labels,
                                                      const int* __restrict__ inverse,
                                                      T* __restrict__ dh, long long tokens, int D) {
  const int ns = *splits;
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int r = inverse[t];
    const float4* s = reinterpret_cast<const float4*>(src + static_cast<long long>(r < 0 ? 0 : r) * D);
    const float c = r < 0 || scale == nullptr ? 1.f : scale[r];
    const float own = r < 0 ? 0.f : gout[t] * inv_temp * label_grad[r];
    const uint2* wr = own != 0.f ? reinterpret_cast<const uint2*>(w + labels[t] * ldw) : nullptr;
    for (int i = threadIdx.x; i < D / 4; i += blockDim.x) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= 0) {
        v = s[i];
        for (int k = 1; k < ns; ++k) {
          const float4 a = s[i + k * (split_stride / 4)];
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
        }
        v.x *= c; v.y *= c; v.z *= c; v.w *= c;
        if (wr != nullptr) {
          const float2 a = unpack_bf16x2(wr[i].x), b = unpack_bf16x2(wr[i].y);
          v.x = fmaf(own, a.x, v.x);
          v.y = fmaf(own, a.y, v.y);
          v.z = fmaf(own, b.x, v.z);
          v.w = fmaf(own, b.y, v.w);
        }
      }
      if (sizeof(T) == 2)
        reinterpret_cast<uint2*>(dh + t * D)[i] = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      else
        reinterpret_cast<float4*>(dh + t * D)[i] = v;
    }
  }
}

__device__ __forceinline__ void unpack8(uint4 u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = unpack_bf16x2(w[j]);
    x[2 * j] = a.x;
    x[2 * j + 1] = a.y;
  }
}
// The labels' part of dW, which the product's epilogue adds in fp32: for every label v, the sum
// over its tokens of their entry of G times their hidden row. The block at a label's first token
// (and, in y, at eight columns a thread) adds up that label's rows in token order: no atomics.
// SORTED: tokens come sorted by label (stable), so a label's are neighbours; otherwise every
// block looks through all labels, which for up to kLabelScanTokens tokens costs less than the
// sort's launches, or little more (us without and with the sort, its launches included:
// D = 256: 13 and 34 for 1024 tokens, 23 and 39 for 2048, 51 and 48 for 4096, 134 and 84 for 8192;
// D = 1024: 26 and 37, 56 and 50, 142 and 86 for 2048, 4096 and 8192; D = 2048: 36 and 39, 90 and
// 53, 250 and 121, where the products of 4096 tokens take a millisecond). Rows and entries are listed a block's width at a time, so that the row loads
// do not wait for them, and eight rows are fetched at once. Bound by latency: the chain of loads
// that leads to a row and the longest run (16384 tokens, 300 of them with one label, D = 1024:
// 90 us; 149 with four columns a thread and the rows' loads left to the compiler).
template <bool SORTED>
__global__ void __launch_bounds__(128) label_rows_kernel(const int* __restrict__ sorted,
                                                         const int64_t* __restrict__ token,
                                                         const int64_t* __restrict__ labels,
                                                         const int* __restrict__ inverse,
                                                         const float* __restrict__ label_grad,
                                                         const float* __restrict__ gout, float inv_temp,
                                                         const __nv_bfloat16* __restrict__ h, int D,
                                                         float* __restrict__ sums, int* __restrict__ row_of,
                                                         int tokens) {
  __shared__ int s_row[128], s_warp[4];
  __shared__ float s_f[128];
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;  // this thread's first column
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, step = blockDim.x;
  for (int i = blockIdx.x; i < tokens; i += gridDim.x) {
    const long long v = SORTED ? sorted[i] : labels[i];
    // a label left out (ignored or outside the vocabulary) is left out for all its tokens
    if (inverse[SORTED ? token[i] : i] < 0) continue;
    if (SORTED) {
      if (i > 0 && sorted[i - 1] == v) continue;
    } else {
      bool earlier = false;
#pragma unroll 8
      for (int j = threadIdx.x; j < i; j += step) earlier |= labels[j] == v;
      if (__syncthreads_or(earlier)) continue;
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) row_of[v] = i;
    float s[8] = {};
    for (int j0 = i; j0 < tokens; j0 += step) {
      const int j = j0 + threadIdx.x;
      const bool mine = j < tokens && (SORTED ? sorted[j] == v : labels[j] == v);
      int at = threadIdx.x;
      if (!SORTED) {  // the place among the block's matches
        const unsigned all = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) s_warp[warp] = __popc(all);
        __syncthreads();
        at = __popc(all & ((1u << lane) - 1u));
        for (int k = 0; k < warp; ++k) at += s_warp[k];
      }
      if (mine) {
        const long long t = SORTED ? token[j] : j;
        const int r = inverse[t];
        s_row[at] = r;
        s_f[at] = gout[t] * inv_temp * label_grad[r];
      }
      const int n = __syncthreads_count(mine);
      if (c < D) {
        for (int k0 = 0; k0 < n; k0 += 8) {
          uint4 u[8];  // eight rows on their way at once
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k0 + k < n)
              u[k] = *reinterpret_cast<const uint4*>(h + static_cast<long long>(s_row[k0 + k]) * D + c);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (k0 + k >= n) continue;
            float x[8];
            unpack8(u[k], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = fmaf(s_f[k0 + k], x[e], s[e]);
          }
        }
      }
      __syncthreads();
      if (SORTED && n < step) break;
    }
    if (c >= D) continue;
    float4* p = reinterpret_cast<float4*>(sums + static_cast<long long>(i) * D + c);
    p[0] = make_float4(s[0], s[1], s[2], s[3]);
    p[1] = make_float4(s[4], s[5], s[6], s[7]);
  }
}

CUtensorMap head_map(const void* base, long long rows, long long cols, long long ld, int box_cols, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * 2)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_tensor_map(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                                 strides, box, estr,
                                 box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  if (r != CUDA_SUCCESS)
    throw std::runtime_error("linear_token_logprobs: cuTensorMapEncodeTiled failed with code " +
                             std::to_string(r));
  return m;
}

int sm_count() {
  int dev, n;
  PLG_CUDA_CHECK(cudaGetDevice(&dev));
  PLG_CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
  return n;
}

template <bool STATS, bool STORE, bool CAP, bool SEG>
void launch_head(const HeadProblem& p, const HeadArgs& a, void* X, long long ldx, cudaStream_t st) {
  auto kern = head_kernel<STATS, STORE, CAP, SEG>;
  set_max_smem_once(reinterpret_cast<const void*>(kern), kSmemBytes);
  if (SEG) {
    // the register split waits forever unless the launch owns what the epilogue asks for
    static const int regs = [&] {
      cudaFuncAttributes f;
      PLG_CUDA_CHECK(cudaFuncGetAttributes(&f, kern));
      return f.numRegs;
    }();
    if (kLoadRegs * 128 + kEpiRegs * 32 * kEpiWarps > regs * kThreads)
      throw std::runtime_error("linear_token_logprobs: the kernel was built with too few registers");
  }
  const CUtensorMap ta = head_map(p.h, p.rows, p.D, p.ldh, kBK, kBM);
  const CUtensorMap tb = head_map(p.w, p.N, p.D, p.ldw, kBK, a.bn / 2);
  const CUtensorMap tx = STORE ? head_map(X, p.rows, p.N, ldx, 32, 32) : ta;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const long long work = static_cast<long long>((p.rows + 2 * kBM - 1) / (2 * kBM)) * a.n_tiles;
  const int pairs = static_cast<int>(std::min<long long>(work, head_pairs()));
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  PLG_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, tx, a));
}

template <bool STATS, bool STORE>
void dispatch_head(const HeadProblem& p, const HeadArgs& a, void* X, long long ldx, cudaStream_t st) {
  const bool cap = p.softcap > 0.f;
  if (STATS && a.segs > 1) {
    if (cap) launch_head<STATS, STORE, true, STATS>(p, a, X, ldx, st);
    else launch_head<STATS, STORE, false, STATS>(p, a, X, ldx, st);
  } else {
    if (cap) launch_head<STATS, STORE, true, false>(p, a, X, ldx, st);
    else launch_head<STATS, STORE, false, false>(p, a, X, ldx, st);
  }
}

template <int NT, bool CAP>
void launch_thin(const HeadProblem& p, const ThinArgs& a, int ctas, cudaStream_t st) {
  auto kern = thin_kernel<NT, CAP>;
  set_max_smem_once(reinterpret_cast<const void*>(kern), Thin<NT>::kSmem);
  const CUtensorMap tw = head_map(p.w, p.N, p.D, p.ldw, kBK, a.tile);
  const CUtensorMap th = head_map(p.h, p.rows, p.D, p.ldh, kBK, NT);
  kern<<<ctas, kThinThreads, Thin<NT>::kSmem, st>>>(tw, th, a);
  PLG_CUDA_CHECK(cudaGetLastError());
}

template <int NT>
void dispatch_thin(const HeadProblem& p, const ThinArgs& a, int ctas, cudaStream_t st) {
  if (p.softcap > 0.f) launch_thin<NT, true>(p, a, ctas, st);
  else launch_thin<NT, false>(p, a, ctas, st);
}

void check_x(const void* X, long long ldx) {
  if (ldx % 8 || (reinterpret_cast<uintptr_t>(X) & 15))
    throw std::invalid_argument("linear_token_logprobs: the gradient rows must be 16-byte aligned");
}

void check_head(const HeadProblem& p) {
  if (p.D <= 0 || p.D % 8 || p.ldh % 8 || p.ldw % 8)
    throw std::invalid_argument("linear_token_logprobs: D and the row strides must be multiples of 8");
  if ((reinterpret_cast<uintptr_t>(p.h) | reinterpret_cast<uintptr_t>(p.w)) & 15)
    throw std::invalid_argument("linear_token_logprobs: hidden and weight must be 16-byte aligned");
  if (p.N <= 0) throw std::invalid_argument("linear_token_logprobs: an empty vocabulary");
}

HeadArgs base_args(const HeadProblem& p) {
  HeadArgs a{};
  a.rows = p.rows;
  a.N = p.N;
  a.k_blocks = (p.D + kBK - 1) / kBK;
  a.segs = (a.k_blocks + kSegBlocks - 1) / kSegBlocks;
  a.bn = p.bn;
  a.n_tiles = (p.N + a.bn - 1) / a.bn;
  // the rows of a group of m tiles take at most 32 MB of L2
  const long long tile_bytes = 2LL * kBM * p.D * 2;
  a.group_m = static_cast<int>(std::max<long long>(1, (32LL << 20) / tile_bytes));
  a.n_rows = p.n_rows;
  a.row_map = p.row_map;
  a.labels = p.labels;
  a.label0 = p.label0;
  a.k = kLog2e / p.temperature;
  a.cap = p.softcap;
  a.inv_cap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;
  a.status = p.status;
  return a;
}

}  // namespace

int head_pairs() { return sm_count() / 2; }

// Columns of a tile: the width whose last wave over the CTA pairs is fullest. A 256-wide
// tile reuses the hidden rows most, so a narrower one has to save more than 1/64 of the
// columns walked.
int head_tile_n(int rows, int N) {
  const int pairs = head_pairs();
  const long long m_tiles = (rows + 2 * kBM - 1) / (2 * kBM);
  int best = kMaxBN;
  double best_cost = 0;
  for (int bn = kMaxBN; bn >= 128; bn -= 32) {
    const long long units = m_tiles * ((N + bn - 1) / bn);
    const double cost = static_cast<double>((units + pairs - 1) / pairs) * bn * (bn == kMaxBN ? 1.0 : 1.0 + 1.0 / 64);
    if (bn == kMaxBN || cost < best_cost) {
      best = bn;
      best_cost = cost;
    }
  }
  return best;
}

// CTAs of the few-rows kernel: one per SM, each with at least 32 entries
static int thin_ctas(int V) { return std::max(1, std::min(sm_count(), V / 32)); }

bool head_is_thin(const HeadProblem& p) { return p.n_rows == nullptr && p.rows <= kThinRows; }

int head_parts(const HeadProblem& p) {
  return head_is_thin(p) ? 4 * thin_ctas(p.N) : 2 * ((p.N + p.bn - 1) / p.bn);
}

static void head_thin(const HeadProblem& p, void* part, float* target, cudaStream_t st) {
  const int ctas = thin_ctas(p.N);
  ThinArgs a{};
  a.T = p.rows;
  a.V = p.N;
  const int share = (p.N + ctas - 1) / ctas;  // the largest share of a CTA, in equal tiles
  const int tiles = (share + kThinEntries - 1) / kThinEntries;
  a.tile = (share + tiles - 1) / tiles;
  a.k_blocks = (p.D + kBK - 1) / kBK;
  a.segs = (a.k_blocks + kThinSegBlocks - 1) / kThinSegBlocks;
  a.labels = p.labels;
  a.k = kLog2e / p.temperature;
  a.cap = p.softcap;
  a.inv_cap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;
  a.part = static_cast<float2*>(part);
  a.target = target;
  a.status = p.status;
  if (p.rows <= 32) dispatch_thin<32>(p, a, ctas, st);
  else if (p.rows <= 64) dispatch_thin<64>(p, a, ctas, st);
  else dispatch_thin<128>(p, a, ctas, st);
}

void head_stats(const HeadProblem& p, void* part, float* target, const float* ref, void* X, long long ldx,
                cudaStream_t st) {
  if (p.rows <= 0) return;
  check_head(p);
  if (head_is_thin(p) && X == nullptr) return head_thin(p, part, target, st);
  HeadArgs a = base_args(p);
  a.part = static_cast<float2*>(part);
  a.target = target;
  if (X != nullptr) {
    check_x(X, ldx);
    a.ref = ref;
    dispatch_head<true, true>(p, a, X, ldx, st);
  } else {
    dispatch_head<true, false>(p, a, nullptr, 0, st);
  }
}

void head_join(const HeadProblem& p, const void* part, const float* target, long long V,
               long long ignore_index, float* out, const float* ref, float* lse2, float* label_grad,
               int* flag, cudaStream_t st) {
  if (p.rows <= 0) return;
  const int parts = head_parts(p);
  const float2* pp = static_cast<const float2*>(part);
  const float k = kLog2e / p.temperature;
  // a warp per row fills the machine from about 148 * 8 rows on
  const bool many = p.rows >= 1024;
  launch_dependent(many ? join_kernel<1> : join_kernel<8>, many ? std::min((p.rows + 7) / 8, 148 * 8) : p.rows, 256,
                   st, pp, parts, p.rows, p.n_rows, p.row_map, p.labels, V, ignore_index, target, k, p.softcap, out,
                   ref, lse2, label_grad, flag);
}

void head_recompute(const HeadProblem& p, const float* lse2, const float* gout, const int* only_if, void* X,
                    long long ldx, cudaStream_t st) {
  if (p.rows <= 0) return;
  check_head(p);
  check_x(X, ldx);
  HeadArgs a = base_args(p);
  a.ref = lse2;
  a.gout = gout;
  a.inv_temp = 1.f / p.temperature;
  a.only_if = only_if;
  dispatch_head<false, true>(p, a, X, ldx, st);
}

void head_scale_rows(const HeadProblem& p, const float* lse2, const float* ref, const float* gout, void* X,
                     long long ldx, float* scale, void* hs, cudaStream_t st) {
  if (p.rows <= 0) return;
  if (p.ldh != p.D || p.D % 8)
    throw std::invalid_argument("linear_token_logprobs: packed rows of a multiple of 8 columns");
  scale_rows_kernel<<<std::min(p.rows, 148 * 16), 128, 0, st>>>(
      static_cast<const __nv_bfloat16*>(p.h), p.D, p.row_map, p.n_rows, p.labels, lse2, ref, gout, 1.f / p.temperature,
      static_cast<__nv_bfloat16*>(X), ldx, scale, static_cast<__nv_bfloat16*>(hs), p.rows);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_compact(const int64_t* labels, long long T, long long V, long long ignore_index, int* row_map,
                  int* inverse, int* count, float* out, cudaStream_t st) {
  if (T <= 0) return;
  compact_kernel<<<static_cast<unsigned>((T + kScan - 1) / kScan), kScan, 0, st>>>(
      labels, T, V, ignore_index, row_map, inverse, count, out);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_gather(const HeadProblem& p, const void* h, bool fp32, long long ldh, void* out, int cap_rows,
                 float* ref, cudaStream_t st) {
  if (cap_rows <= 0) return;
  const int D = p.D;
  if (D % 8 || ldh % 8 || p.ldw % 8 ||
      ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(p.w)) & 15))
    throw std::invalid_argument("linear_token_logprobs: D and the row strides must be multiples of 8, "
                                "rows 16-byte aligned");
  const int blocks = std::min(cap_rows, 148 * 16);
  const float k = kLog2e / p.temperature;
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(p.w);
  if (fp32)
    gather_kernel<float><<<blocks, 128, 0, st>>>(static_cast<const float*>(h), ldh, D, p.row_map, p.n_rows,
                                                 static_cast<__nv_bfloat16*>(out), cap_rows, w, p.ldw, p.labels, k,
                                                 p.softcap, ref);
  else
    gather_kernel<__nv_bfloat16><<<blocks, 128, 0, st>>>(static_cast<const __nv_bfloat16*>(h), ldh, D, p.row_map,
                                                         p.n_rows, static_cast<__nv_bfloat16*>(out), cap_rows, w,
                                                         p.ldw, p.labels, k, p.softcap, ref);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_label_rows(const HeadProblem& p, const int* sorted, const int64_t* token, const int* inverse,
                     const float* label_grad, const float* gout, float* sums, int* row_of, int tokens,
                     cudaStream_t st) {
  PLG_CUDA_CHECK(cudaMemsetAsync(row_of, 0xff, sizeof(int) * static_cast<size_t>(p.N), st));
  if (tokens <= 0) return;
  // the search through all labels takes whole blocks
  const int threads = sorted == nullptr ? 128 : std::min(128, (p.D / 8 + 31) / 32 * 32);
  const dim3 grid(std::min(tokens, 148 * 16), (p.D / 8 + threads - 1) / threads);
  auto kern = sorted != nullptr ? label_rows_kernel<true> : label_rows_kernel<false>;
  kern<<<grid, threads, 0, st>>>(sorted, token, p.labels, inverse, label_grad, gout, 1.f / p.temperature,
                                 static_cast<const __nv_bfloat16*>(p.h), p.D, sums, row_of, tokens);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_scatter(const HeadProblem& p, const float* src, long long split_stride, const int* splits,
                  const float* scale, const float* label_grad, const float* gout, const int* inverse, void* dh,
                  bool fp32, long long tokens, cudaStream_t st) {
  if (tokens <= 0) return;
  const int blocks = static_cast<int>(std::min<long long>(tokens, 148 * 16));
  auto run = [&](auto kern, auto* out) {
    kern<<<blocks, 256, 0, st>>>(src, split_stride, splits, scale, label_grad, gout, 1.f / p.temperature,
                                 static_cast<const __nv_bfloat16*>(p.w), p.ldw, p.labels, inverse, out, tokens,
                                 p.D);
  };
  if (fp32) run(scatter_kernel<float>, static_cast<float*>(dh));
  else run(scatter_kernel<__nv_bfloat16>, static_cast<__nv_bfloat16*>(dh));
  PLG_CUDA_CHECK(cudaGetLastError());
}

}  // namespace plg
