// Log-probabilities of given tokens under a linear head, and their gradient.
//
//   a[t, v]  = <h_t, w_v>                       tcgen05 product, fp32 accumulators
//   z[t, v]  = softcap(a) / temperature         softcap(a) = cap * tanh(a / cap), or a
//   out[t]   = z[t, y_t] - log sum_v exp z[t, v]
//   dout/dz  = onehot(y_t) - softmax(z_t)
//
// The logits never reach memory in the forward pass: the product's epilogue turns each
// accumulator row of a tile into a running (reference, sum of 2^(z log2e - reference))
// pair, and a second small kernel joins a row's pairs in a fixed order. The gradient pass
// recomputes the tile and stores bf16 G = g_t * dout/dz, the operand of the two gradient
// products (dh = G W, dW = G^T h, gemm_tcgen05.cu).
//
// Rows whose label is ignore_index are left out of the products: compact_rows lists the
// others on the device, gather_rows packs their hidden rows, and every later kernel reads
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
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kMaxStageBytes = kABytes + (kMaxBN / 2) * kBK * 2;
constexpr int kSmemBytes = kStages * kMaxStageBytes + 1024 + 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum HeadMode { kStats = 0, kGrad = 1 };

struct HeadArgs {
  int rows, N, k_blocks;
  int bn, m_tiles, n_tiles, group_m;
  const int* n_rows;            // device row count (null: rows)
  const int* row_map;           // compact row -> token (null: identity)
  const int64_t* labels;        // per token
  long long label0;             // vocabulary index of column 0
  float k;                      // log2(e) / temperature
  float cap, inv_cap;
  int* status;
  float2* part;                 // stats: [rows][2 * n_tiles]
  float* target;                // stats: [rows] accumulator (after the softcap) of the label
  const float* lse2;            // grad: [rows] log2 of the sum of 2^(z log2e)
  const float* gout;            // grad: per token
  float inv_temp;
  __nv_bfloat16* G;
  long long ldg;
};

__device__ __forceinline__ float ex2(float x) { return fast_exp2(x); }

// Persistent CTA-pair kernel: 256 x bn tiles with tcgen05.mma.cta_group::2. CTA rank r
// holds rows [128 r, 128 r + 128) of the tile and loads those of A and half of B's bn
// columns. Warp 0 loads (TMA), warp 1 of rank 0 issues the MMAs, 8 warps per CTA drain the
// accumulator (two warps per 32-row quadrant, alternate 32-column chunks), double
// buffered in TMEM against the next tile's main loop.
template <int MODE, bool CAP>
__global__ void __launch_bounds__(kThreads, 1)
    head_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const HeadArgs args) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kStages * kMaxStageBytes);
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
      for (int w = pair; w < total && ok; w += npairs, ++local) {
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
        for (int kb = 0; kb < args.k_blocks; ++kb) {
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
                           (kb > 0 || kk > 0) ? 1u : 0u);
          tc_commit_pair(&empty_bar[stage], 0x3);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit_pair(&accf_bar[buf], 0x3);
      }
      if (!ok) *abort_flag = 1;
      tc_commit_pair(done_bar, 0x3);
    }
    if (lane == 0 && !mbar_wait_bounded(done_bar, 0, nullptr)) record_status(args.status, kTimeoutDrain);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;           // TMEM lane quadrant this warp may access
    const int half = (warp - 2) >> 2;  // which of the quadrant's two warps
    const int row_in_tile = q * 32 + lane;
    const int chunks = bn / 32;
    int local = 0;
    for (int w = pair; w < total; w += npairs, ++local) {
      int mt, nt;
      decode(w, mt, nt);
      const int buf = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      const int row = mt * 2 * kBM + static_cast<int>(rank) * kBM + row_in_tile;
      const bool live = row < rows;
      // this row's label as a column of this launch, and its factors
      long long lab = -1;
      float lse2 = 0.f, coef = 0.f;
      if (live) {
        const int tok = args.row_map != nullptr ? args.row_map[row] : row;
        lab = args.labels[tok] - args.label0;
        if (MODE == kGrad) {
          lse2 = args.lse2[row];
          coef = args.gout[tok] * args.inv_temp;
        }
      }
      if (!mbar_wait_bounded(&accf_bar[buf], acc_phase, abort_flag)) {
        record_status(args.status, kTimeoutAccFull);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buf * kMaxBN;
      const bool warp_live = row - lane < rows;  // any live row in this warp
      if (MODE == kStats ? warp_live : row - lane < args.rows) {
        float ref = -INFINITY, s0 = 0.f, s1 = 0.f;
#pragma unroll 1
        for (int c = half; c < chunks; c += 2) {
          uint32_t r[32];
          __syncwarp();
          tmem_ld_32x32b_x32(t_row + c * 32, r);
          tmem_ld_wait();
          const int col0 = nt * bn + c * 32;
          if (col0 >= args.N) continue;  // uniform over the grid's columns
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] = __uint_as_float(r[i]);
            if (CAP && MODE == kStats) v[i] = args.cap * tanhf(v[i] * args.inv_cap);
          }
          const int lc = (lab >= col0 && lab < col0 + 32) ? static_cast<int>(lab - col0) : -1;
          if (MODE == kStats) {
            if (lc >= 0) {
              float y = 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i == lc) y = v[i];
              if (col0 + lc < args.N) args.target[row] = y;
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
              fadd2(s0, s1, s0, s1, ex2(e0), ex2(e1));
            }
          } else {
            uint32_t o[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float a0 = v[i], a1 = v[i + 1], d0 = coef, d1 = coef;
              if (CAP) {
                const float t0 = tanhf(a0 * args.inv_cap), t1 = tanhf(a1 * args.inv_cap);
                a0 = args.cap * t0;
                a1 = args.cap * t1;
                d0 *= 1.f - t0 * t0;
                d1 *= 1.f - t1 * t1;
              }
              float e0, e1;
              ffma2(e0, e1, a0, a1, args.k, args.k, -lse2, -lse2);
              float g0 = -ex2(e0), g1 = -ex2(e1);
              if (i == lc) g0 += 1.f;
              if (i + 1 == lc) g1 += 1.f;
              o[i / 2] = pack_bf16x2(g0 * d0, g1 * d1);
            }
            // rows past the count up to the tile's end are the products' zero padding
            if (!live) {
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0u;
            }
            if (row < args.rows) {
              __nv_bfloat16* gp = args.G + row * args.ldg + col0;
              if (col0 + 32 <= args.N) {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                  *reinterpret_cast<uint4*>(gp + 2 * i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (col0 + i < args.N) {
                    const uint32_t u = (i & 1) ? (o[i / 2] >> 16) : (o[i / 2] & 0xffffu);
                    reinterpret_cast<uint16_t*>(gp)[i] = static_cast<uint16_t>(u);
                  }
              }
            }
          }
        }
        if (MODE == kStats && live)
          args.part[static_cast<long long>(row) * (2 * args.n_tiles) + 2 * nt + half] =
              make_float2(ref, s0 + s1);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(&acce_bar[buf], 0);
    }
  }

  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- small kernels
constexpr int kScan = 1024;

// Block b lists the kept tokens of [1024 b, 1024 b + 1024): row_map (compact -> token, in
// token order), inverse (token -> compact or -1); ignored tokens get out = 0, labels
// outside the vocabulary NaN (and no gradient). The block counts the kept tokens before
// its own range itself, so one launch does the scan; the last block writes the total.
__global__ void __launch_bounds__(kScan) compact_kernel(const int64_t* __restrict__ labels, long long T,
                                                        long long V, long long ignore_index,
                                                        int* __restrict__ row_map,
                                                        int* __restrict__ inverse,
                                                        int* __restrict__ count,
                                                        float* __restrict__ out) {
  __shared__ int s_warp[32];
  __shared__ int s_base;
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

// packed bf16 hidden rows of the kept tokens; zero rows up to the next multiple of 256
template <typename T>
__global__ void __launch_bounds__(256) gather_kernel(const T* __restrict__ h, long long ldh, int D,
                                                     const int* __restrict__ row_map,
                                                     const int* __restrict__ count,
                                                     __nv_bfloat16* __restrict__ out, int cap_rows) {
  const int n = *count;
  const int pad = min(cap_rows, (n + 255) / 256 * 256);
  for (int r = blockIdx.x; r < pad; r += gridDim.x) {
    uint4* dst = reinterpret_cast<uint4*>(out + static_cast<long long>(r) * D);
    if (r >= n) {
      for (int i = threadIdx.x; i < D / 8; i += blockDim.x) dst[i] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const T* src = h + static_cast<long long>(row_map[r]) * ldh;
    for (int i = threadIdx.x; i < D / 8; i += blockDim.x) {
      if (sizeof(T) == 2) {
        dst[i] = reinterpret_cast<const uint4*>(src)[i];
      } else {
        const float4 a = reinterpret_cast<const float4*>(src)[2 * i];
        const float4 b = reinterpret_cast<const float4*>(src)[2 * i + 1];
        dst[i] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y),
                            pack_bf16x2(b.z, b.w));
      }
    }
  }
}

// One warp per row joins the row's (reference, sum) pairs (lane-strided, then a fixed
// shuffle tree: the same order every run) and writes out = z_label - lse.
__global__ void __launch_bounds__(256) join_kernel(const float2* __restrict__ part, int parts, int rows_,
                                                   const int* __restrict__ n_rows,
                                                   const int* __restrict__ row_map,
                                                   const int64_t* __restrict__ labels, long long V,
                                                   long long ignore_index,
                                                   const float* __restrict__ target, float k,
                                                   float* __restrict__ out, float* __restrict__ lse2) {
  const int lane = threadIdx.x & 31;
  const int nw = gridDim.x * (blockDim.x >> 5);
  const int rows = n_rows != nullptr ? min(*n_rows, rows_) : rows_;
  for (int row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); row < rows; row += nw) {
    const float2* p = part + static_cast<long long>(row) * parts;
    float m = -INFINITY, s = 0.f;
    for (int i = lane; i < parts; i += 32) {
      const float2 v = p[i];
      const float nm = fmaxf(m, v.x), sub = nm == -INFINITY ? 0.f : nm;
      s = s * ex2(m - sub) + v.y * ex2(v.x - sub);
      m = nm;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, o);
      const float os = __shfl_xor_sync(0xffffffffu, s, o);
      const float nm = fmaxf(m, om), sub = nm == -INFINITY ? 0.f : nm;
      s = s * ex2(m - sub) + os * ex2(om - sub);
      m = nm;
    }
    if (lane == 0) {
      const int tok = row_map != nullptr ? row_map[row] : row;
      const int64_t y = labels[tok];
      const float l2 = log2f(s);
      float v = 0.f;
      if (y != ignore_index)
        v = (y >= 0 && y < V) ? kLn2 * (fmaf(target[row], k, -m) - l2) : __int_as_float(0x7fc00000);
      out[tok] = v;
      if (lse2 != nullptr) lse2[row] = m + l2;
    }
  }
}

// dh[token] = fp32 compact gradient row in dh's type, zeros for the tokens left out
template <typename T>
__global__ void __launch_bounds__(256) scatter_kernel(const float* __restrict__ src,
                                                      const int* __restrict__ inverse,
                                                      T* __restrict__ dh, long long tokens, int D) {
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int r = inverse[t];
    const float4* s = reinterpret_cast<const float4*>(src + static_cast<long long>(r < 0 ? 0 : r) * D);
    for (int i = threadIdx.x; i < D / 4; i += blockDim.x) {
      const float4 v = r < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : s[i];
      if (sizeof(T) == 2)
        reinterpret_cast<uint2*>(dh + t * D)[i] = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
      else
        reinterpret_cast<float4*>(dh + t * D)[i] = v;
    }
  }
}

CUtensorMap head_map(const void* base, long long rows, long long cols, long long ld, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * 2)};
  cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_tensor_map(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                                 strides, box, estr, CU_TENSOR_MAP_SWIZZLE_128B);
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

template <int MODE, bool CAP>
void launch_head(const HeadProblem& p, HeadArgs a, cudaStream_t st) {
  auto kern = head_kernel<MODE, CAP>;
  set_max_smem_once(reinterpret_cast<const void*>(kern), kSmemBytes);
  const CUtensorMap ta = head_map(p.h, p.rows, p.D, p.ldh, kBM);
  const CUtensorMap tb = head_map(p.w, p.N, p.D, p.ldw, a.bn / 2);
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
  const long long work = static_cast<long long>(a.m_tiles) * a.n_tiles;
  const int pairs = static_cast<int>(std::min<long long>(work, head_pairs()));
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  PLG_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, a));
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
  a.bn = p.bn;
  a.m_tiles = (p.rows + 2 * kBM - 1) / (2 * kBM);
  a.n_tiles = (p.N + a.bn - 1) / a.bn;
  // the rows of a group of m tiles take at most 32 MB of L2
  const long long tile_bytes = 2LL * kBM * p.D * 2;
  a.group_m = static_cast<int>(std::max<long long>(1, (32LL << 20) / tile_bytes));
  a.n_rows = p.n_rows;
  a.row_map = p.row_map;
  a.labels = p.labels;
  a.label0 = p.label0;
  a.k = kLog2e / p.temperature;
  a.inv_temp = 1.f / p.temperature;
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

void head_stats(const HeadProblem& p, void* part, float* target, cudaStream_t st) {
  if (p.rows <= 0) return;
  check_head(p);
  HeadArgs a = base_args(p);
  a.part = static_cast<float2*>(part);
  a.target = target;
  if (p.softcap > 0.f) launch_head<kStats, true>(p, a, st);
  else launch_head<kStats, false>(p, a, st);
}

void head_join(const HeadProblem& p, const void* part, const float* target, long long V,
               long long ignore_index, float* out, float* lse2, cudaStream_t st) {
  if (p.rows <= 0) return;
  const int parts = 2 * ((p.N + p.bn - 1) / p.bn);
  const int blocks = std::min((p.rows + 7) / 8, 148 * 8);
  join_kernel<<<blocks, 256, 0, st>>>(static_cast<const float2*>(part), parts, p.rows, p.n_rows, p.row_map,
                                      p.labels, V, ignore_index, target, kLog2e / p.temperature, out, lse2);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_grad(const HeadProblem& p, const float* lse2, const float* gout, void* G, long long ldg,
               cudaStream_t st) {
  if (p.rows <= 0) return;
  check_head(p);
  if (ldg % 8 || (reinterpret_cast<uintptr_t>(G) & 15))
    throw std::invalid_argument("linear_token_logprobs: the gradient rows must be 16-byte aligned");
  HeadArgs a = base_args(p);
  a.lse2 = lse2;
  a.gout = gout;
  a.G = static_cast<__nv_bfloat16*>(G);
  a.ldg = ldg;
  if (p.softcap > 0.f) launch_head<kGrad, true>(p, a, st);
  else launch_head<kGrad, false>(p, a, st);
}

void head_compact(const int64_t* labels, long long T, long long V, long long ignore_index, int* row_map,
                  int* inverse, int* count, float* out, cudaStream_t st) {
  if (T <= 0) return;
  compact_kernel<<<static_cast<unsigned>((T + kScan - 1) / kScan), kScan, 0, st>>>(
      labels, T, V, ignore_index, row_map, inverse, count, out);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_gather(const void* h, bool fp32, long long ldh, int D, const int* row_map, const int* count,
                 void* out, int cap_rows, cudaStream_t st) {
  if (cap_rows <= 0) return;
  if (D % 8 || ldh % 8 || ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(out)) & 15))
    throw std::invalid_argument("linear_token_logprobs: D and hidden's row stride must be multiples of 8, "
                                "rows 16-byte aligned");
  const int blocks = std::min(cap_rows, 148 * 16);
  if (fp32)
    gather_kernel<float><<<blocks, 256, 0, st>>>(static_cast<const float*>(h), ldh, D, row_map, count,
                                                 static_cast<__nv_bfloat16*>(out), cap_rows);
  else
    gather_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(h), ldh, D,
                                                         row_map, count,
                                                         static_cast<__nv_bfloat16*>(out), cap_rows);
  PLG_CUDA_CHECK(cudaGetLastError());
}

void head_scatter(const float* src, const int* inverse, void* dh, bool fp32, long long tokens, int D,
                  cudaStream_t st) {
  if (tokens <= 0) return;
  const int blocks = static_cast<int>(std::min<long long>(tokens, 148 * 16));
  if (fp32)
    scatter_kernel<float><<<blocks, 256, 0, st>>>(src, inverse, static_cast<float*>(dh), tokens, D);
  else
    scatter_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(src, inverse, static_cast<__nv_bfloat16*>(dh),
                                                          tokens, D);
  PLG_CUDA_CHECK(cudaGetLastError());
}

}  // namespace plg
