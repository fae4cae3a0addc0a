// Losses over per-token log-probabilities (paired preference loss, clipped policy loss with
// a KL term) and over MoE router logits (balance and z loss), forward and backward.
//
// All of them stream their inputs and are bound by memory, or, at a few thousand tokens, by
// the host: a forward and backward of one to four launches takes it 70 to 80 us, the GPU 10
// to 16. Every sum runs in a fixed order: per-warp or per-block partial sums go to a
// workspace and one block joins them, so results repeat bit for bit. Masked places are
// skipped by selection, never by a product with 0, so that whatever they hold (infinities,
// NaN) reaches neither a loss nor a gradient.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "common.cuh"
#include "ops.h"

namespace plg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Tokens of one row that a warp takes at a time: 1024 once that gives every warp of the
// machine (148 SMs x 16) a unit, fewer, down to 128, where there would be too few of them
// (policy loss of 8 rows of 1023 tokens: 17.9 us at 1024, 6.4 us at 128).
constexpr int kMaxWarpTokens = 1024, kMinWarpTokens = 128;

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int VEC>
__device__ __forceinline__ void load_f(const float* p, float (&v)[VEC]) {
  if (VEC == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    v[0] = *p;
  }
}

// VEC values at element `i` of an fp32 or bf16 row
template <int VEC>
__device__ __forceinline__ void load_any(const void* p, bool bf16, long long i, float (&v)[VEC]) {
  if (!bf16) {
    load_f<VEC>(static_cast<const float*>(p) + i, v);
  } else if (VEC == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p) + i);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  } else {
    v[0] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  }
}

template <int VEC>
__device__ __forceinline__ void load_mask(const uint8_t* p, bool (&m)[VEC]) {
  if (VEC == 4) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int j = 0; j < VEC; ++j) m[j] = ((u >> (8 * j)) & 0xffu) != 0;
  } else {
    m[0] = *p != 0;
  }
}

// ------------------------------------------------------------------ preference loss
// Row r = side * P + pair of [2, P, S] tensors. A warp sums up to kMaxWarpTokens of a row, so that
// few long rows fill the machine as many short ones do; the pairs are joined apart because the
// loss needs both sides of a pair. Bound by memory: 9 bytes a token with an fp32 reference (511
// pairs of 8192 tokens, bf16 reference: 59 MB in 21 us, 2.8 TB/s; a lane's step loads 4 tokens, 4
// to 16 bytes of each input).
template <int VEC>
__global__ void __launch_bounds__(256) pref_sums_kernel(const PrefArgs a, float2* __restrict__ part,
                                                        int chunks, int len, unsigned* __restrict__ ticket) {
  dependents_may_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  const int lane = threadIdx.x & 31;
  const long long units = 2LL * a.P * chunks;
  const long long nw = static_cast<long long>(gridDim.x) * 8;
  for (long long u = blockIdx.x * 8LL + (threadIdx.x >> 5); u < units; u += nw) {
    const long long r = u / chunks;
    const int t0 = static_cast<int>(u - r * chunks) * len;
    const int t1 = min(a.S, t0 + len);
    const int side = r >= a.P ? 1 : 0;
    const long long pair = r - static_cast<long long>(side) * a.P;
    const float* lp = a.logps + side * a.lp_side + pair * a.lp_pair;
    const long long ro = side * a.ref_side + pair * a.ref_pair;
    const uint8_t* mk = a.mask + side * a.mk_side + pair * a.mk_pair;
    float s = 0.f;
    int n = 0;
#pragma unroll 4
    for (int t = t0 + lane * VEC; t < t1; t += 32 * VEC) {
      float x[VEC], y[VEC];
      bool m[VEC];
      load_f<VEC>(lp + t, x);
      load_mask<VEC>(mk + t, m);
      if (a.ref != nullptr) {
        load_any<VEC>(a.ref, a.ref_bf16, ro + t, y);
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] -= y[j];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        s += m[j] ? x[j] : 0.f;
        n += m[j] ? 1 : 0;
      }
    }
    s = warp_sum(s);
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) part[u] = make_float2(s, __int_as_float(n));
  }
}

// One warp per pair joins its chunks; the last block sums the blocks' losses.
//   h = s_0 - s_1;  sigmoid: (1 - eps) softplus(-b h) + eps softplus(b h);
//   hinge: max(0, 1 - b h);  ipo: (h - 1 / (2 b))^2
// The sums and their difference are taken in 64 bits: h is what is left of sums of thousands of
// tokens. Bound by latency (the chain of a pair and the ticket: 6.7 us for two pairs).
__global__ void __launch_bounds__(256) pref_pairs_kernel(const PrefArgs a, const float2* __restrict__ part,
                                                         int chunks, double* __restrict__ block_loss,
                                                         unsigned* __restrict__ ticket,
                                                         float* __restrict__ row_scale,
                                                         float* __restrict__ loss,
                                                         float* __restrict__ chosen,
                                                         float* __restrict__ rejected) {
  __shared__ double s_loss[8];
  __shared__ bool s_last;
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double acc = 0.0;
  for (long long i = blockIdx.x * 8LL + warp; i < a.P; i += gridDim.x * 8LL) {
    double s[2];
    float inv[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const float2* p = part + (side * static_cast<long long>(a.P) + i) * chunks;
      double t = 0.0;
      long long n = 0;
      for (int c = lane; c < chunks; c += 32) {
        const float2 v = p[c];
        t += v.x;
        n += __float_as_int(v.y);
      }
      t = warp_sum_d(t);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      inv[side] = a.normalized && n > 1 ? 1.f / static_cast<float>(n) : 1.f;
      s[side] = a.normalized && n > 1 ? t / static_cast<double>(n) : t;
    }
    const float h = static_cast<float>(s[0] - s[1]);
    float l, d;  // loss and dloss / dh
    if (a.kind == 0) {
      const float x = a.beta * h;
      const float soft = log1pf(expf(-fabsf(x)));
      l = (1.f - a.smoothing) * (soft + fmaxf(-x, 0.f));
      if (a.smoothing > 0.f) l += a.smoothing * (soft + fmaxf(x, 0.f));
      // d softplus(-x) = -sigmoid(-x), d softplus(x) = sigmoid(x)
      const float e = expf(-fabsf(x)), r = 1.f / (1.f + e);
      const float sig = x >= 0.f ? r : e * r, sig_neg = x >= 0.f ? e * r : r;
      d = a.beta * (a.smoothing * sig - (1.f - a.smoothing) * sig_neg);
    } else if (a.kind == 1) {
      const float x = 1.f - a.beta * h;
      l = x > 0.f ? x : (x <= 0.f ? 0.f : x);  // NaN stays NaN
      d = x > 0.f ? -a.beta : (x <= 0.f ? 0.f : x);
    } else {
      const float x = h - 0.5f / a.beta;
      l = x * x;
      d = 2.f * x;
    }
    if (lane == 0) {
      const float c = d / static_cast<float>(a.P);
      row_scale[i] = c * inv[0];
      row_scale[a.P + i] = -c * inv[1];
      chosen[i] = static_cast<float>(a.beta * s[0]);
      rejected[i] = static_cast<float>(a.beta * s[1]);
      acc += l;
    }
  }
  if (lane == 0) s_loss[warp] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += s_loss[w];
    block_loss[blockIdx.x] = t;
    __threadfence();
    s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (s_last && warp == 0) {
    __threadfence();
    double t = 0.0;
    for (int b = lane; b < gridDim.x; b += 32) t += static_cast<volatile double*>(block_loss)[b];
    t = warp_sum_d(t);
    if (lane == 0) *loss = static_cast<float>(t / a.P);
  }
}

// grad[r, t] = gout * row_scale[r] where the mask holds, else 0 (contiguous [2, P, S]). Bound by
// its writes (511 pairs of 8192 tokens, 42 MB: 12 us).
template <int VEC>
__global__ void __launch_bounds__(256) pref_grad_kernel(const PrefArgs a, const float* __restrict__ row_scale,
                                                        const float* __restrict__ gout,
                                                        float* __restrict__ grad, int chunks, int len) {
  const int lane = threadIdx.x & 31;
  const long long units = 2LL * a.P * chunks;
  const long long nw = static_cast<long long>(gridDim.x) * 8;
  const float g = *gout;
  for (long long u = blockIdx.x * 8LL + (threadIdx.x >> 5); u < units; u += nw) {
    const long long r = u / chunks;
    const int t0 = static_cast<int>(u - r * chunks) * len;
    const int t1 = min(a.S, t0 + len);
    const int side = r >= a.P ? 1 : 0;
    const uint8_t* mk = a.mask + side * a.mk_side + (r - static_cast<long long>(side) * a.P) * a.mk_pair;
    const float c = g * row_scale[r];
    float* out = grad + r * a.S;
#pragma unroll 4
    for (int t = t0 + lane * VEC; t < t1; t += 32 * VEC) {
      bool m[VEC];
      load_mask<VEC>(mk + t, m);
      if (VEC == 4)
        *reinterpret_cast<float4*>(out + t) =
            make_float4(m[0] ? c : 0.f, m[1 % VEC] ? c : 0.f, m[2 % VEC] ? c : 0.f, m[3 % VEC] ? c : 0.f);
      else
        out[t] = m[0] ? c : 0.f;
    }
  }
}

// ---------------------------------------------------------------------- policy loss
// counts[r] = tokens of row r; block_counts[b] = (tokens, rows with any) of block b's rows.
// A row is counted by one warp, or by the whole block when rows are long. It runs ahead of the
// main pass because a token's gradient needs the counts, and a mask is one byte of a token's 21
// (1024 x 16384: 8 us).
template <bool BLOCK_ROW>
__global__ void __launch_bounds__(256) policy_counts_kernel(const PolicyArgs a, int* __restrict__ counts,
                                                            longlong2* __restrict__ block_counts,
                                                            unsigned* __restrict__ ticket) {
  __shared__ int s_n[8];
  __shared__ long long s_tok[8];
  __shared__ int s_rows[8];
  dependents_may_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = BLOCK_ROW ? threadIdx.x : lane;
  constexpr int kGroup = BLOCK_ROW ? 256 : 32;
  constexpr int kRows = BLOCK_ROW ? 1 : 8;
  long long tokens = 0;
  int rows = 0;
  for (long long r0 = blockIdx.x * static_cast<long long>(kRows); r0 < a.R; r0 += gridDim.x * static_cast<long long>(kRows)) {
    const long long r = r0 + (BLOCK_ROW ? 0 : warp);
    int n = 0;
    if (r < a.R) {
      const uint8_t* mk = a.mask + r * a.mk_row;
      // bytes up to the first 16-byte boundary, 16 at a time, then the rest
      const int head = min(a.S, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(mk) & 15)) & 15));
      const int vecs = (a.S - head) / 16;
      for (int t = sub; t < head; t += kGroup) n += mk[t] != 0;
      const uint4* mv = reinterpret_cast<const uint4*>(mk + head);
#pragma unroll 4
      for (int i = sub; i < vecs; i += kGroup) {
        const uint4 u = mv[i];
        // a bool tensor's bytes are 0 or 1, but any nonzero byte counts once
        n += __popc(__vcmpne4(u.x, 0) & 0x01010101u) + __popc(__vcmpne4(u.y, 0) & 0x01010101u) +
             __popc(__vcmpne4(u.z, 0) & 0x01010101u) + __popc(__vcmpne4(u.w, 0) & 0x01010101u);
      }
      for (int t = head + vecs * 16 + sub; t < a.S; t += kGroup) n += mk[t] != 0;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (BLOCK_ROW) {
      __syncthreads();
      if (lane == 0) s_n[warp] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) n += s_n[w];
    }
    if (r < a.R && (BLOCK_ROW ? threadIdx.x : lane) == 0) {
      counts[r] = n;
      tokens += n;
      rows += n > 0;
    }
  }
  if (lane == 0) {
    s_tok[warp] = tokens;
    s_rows[warp] = rows;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) {
      tokens += s_tok[w];
      rows += s_rows[w];
    }
    block_counts[blockIdx.x] = make_longlong2(tokens, rows);
  }
}

// em1 = e^d - 1 and k3 = e^d - 1 - d, the KL term per token and (its negative) its slope. For
// small d both differences cancel, so the Taylor series is summed there instead (|d| < 1/4:
// the first dropped term is below 2e-8 of the result).
__device__ __forceinline__ void kl_terms(float d, float& em1, float& k3) {
  float p = 1.f / 5040.f;
  p = fmaf(p, d, 1.f / 720.f);
  p = fmaf(p, d, 1.f / 120.f);
  p = fmaf(p, d, 1.f / 24.f);
  p = fmaf(p, d, 1.f / 6.f);
  p = fmaf(p, d, 0.5f);
  const float q = d * d * p, e = expf(d) - 1.f;
  const bool small = fabsf(d) < 0.25f;
  em1 = small ? d + q : e;
  k3 = small ? q : e - d;
}

// Per token, with r = logps - old and d = ref - logps:
//   loss = -A e^r (the bound instead of e^r once A pushes r past it) + kl_coef (e^d - 1 - d)
//   grad = -A e^r (0 past the bound) - kl_coef (e^d - 1)
// each times the token's weight in the mean, known from the counts.
// OLD, REF, ADV: old log-probabilities, reference and per-token advantages are given (a kernel for
// each set: 67 us instead of 80 with the choice made per token). Loss and gradient come from one
// pass, so that nothing is read twice. Bound by memory: 21 bytes a token (1024 x 16384: 352 MB in
// 66 us on one GPU, 5.3 TB/s, 0.81 of the measured copy rate, and in 75 to 78 on another).
constexpr int kPolicyResident = 3;
template <int VEC, bool OLD, bool REF, bool ADV>
__global__ void __launch_bounds__(256, kPolicyResident) policy_kernel(const PolicyArgs a, const int* __restrict__ counts,
                                                     const longlong2* __restrict__ block_counts, int nblocks,
                                                     double* __restrict__ block_sums,
                                                     unsigned* __restrict__ ticket, float* __restrict__ grad,
                                                     float* __restrict__ loss_out, float* __restrict__ kl_out,
                                                     float* __restrict__ clipped_out, int chunks, int len) {
  __shared__ long long s_cnt[2][8];
  __shared__ double s_sum[3][8];
  __shared__ bool s_last;
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long tokens = 0, rows = 0;
  for (int b = threadIdx.x; b < nblocks; b += 256) {
    const longlong2 v = block_counts[b];
    tokens += v.x;
    rows += v.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
  }
  if (lane == 0) {
    s_cnt[0][warp] = tokens;
    s_cnt[1][warp] = rows;
  }
  __syncthreads();
  tokens = rows = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    tokens += s_cnt[0][w];
    rows += s_cnt[1][w];
  }
  const double inv_tokens = 1.0 / static_cast<double>(tokens > 0 ? tokens : 1);
  const double inv_rows = 1.0 / static_cast<double>(rows > 0 ? rows : 1);

  double loss = 0.0, kl = 0.0, clipped = 0.0;
  const long long units = static_cast<long long>(a.R) * chunks;
  const long long nw = static_cast<long long>(gridDim.x) * 8;
  for (long long u = blockIdx.x * 8LL + warp; u < units; u += nw) {
    const long long r = u / chunks;
    const int t0 = static_cast<int>(u - r * chunks) * len;
    const int t1 = min(a.S, t0 + len);
    const float* __restrict__ lp = a.logps + r * a.lp_row;
    const uint8_t* __restrict__ mk = a.mask + r * a.mk_row;
    const float row_adv = ADV ? 0.f : a.adv[r * a.adv_row];
    const float w = static_cast<float>(a.by_sequence ? inv_rows / max(counts[r], 1) : inv_tokens);
    float* __restrict__ gp = grad + r * a.S;
    float sl = 0.f, sk = 0.f;
    int sc = 0;
    float x[VEC], o[VEC], f[VEC], A[VEC];
    bool m[VEC];
    auto fetch = [&](int t) {
      load_f<VEC>(lp + t, x);
      load_mask<VEC>(mk + t, m);
      if (OLD) load_any<VEC>(a.old, a.old_bf16, r * a.old_row + t, o);
      if (REF) load_any<VEC>(a.ref, a.ref_bf16, r * a.ref_row + t, f);
      if (ADV) load_f<VEC>(a.adv + r * a.adv_row + t, A);
    };
    int t = t0 + lane * VEC;
    if (t < t1) fetch(t);
    for (; t < t1; t += 32 * VEC) {
      // this step's values, then the next step's loads ahead of the arithmetic
      float lr[VEC], df[VEC], adv[VEC], g[VEC];
      bool mm[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        lr[j] = OLD ? x[j] - o[j] : 0.f;
        df[j] = REF ? f[j] - x[j] : 0.f;
        adv[j] = ADV ? A[j] : row_adv;
        mm[j] = m[j];
      }
      if (t + 32 * VEC < t1) fetch(t + 32 * VEC);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        // an advantage of 0 gives 0 also where e^r overflows
        const float ratio = OLD ? expf(adv[j] == 0.f && lr[j] > 0.f ? 0.f : lr[j]) : 1.f;
        const bool up = adv[j] > 0.f && lr[j] > a.log_hi, dn = adv[j] < 0.f && lr[j] < a.log_lo;
        const bool clip = up || dn;
        float l = -(up ? a.hi : dn ? a.lo : ratio) * adv[j];
        float d = clip ? 0.f : -adv[j] * ratio;
        if (REF) {
          float em1, k3;
          kl_terms(df[j], em1, k3);
          sk += mm[j] ? k3 : 0.f;
          if (a.kl_coef != 0.f) {  // a KL that is only reported may be infinite
            l = fmaf(a.kl_coef, k3, l);
            d = fmaf(-a.kl_coef, em1, d);
          }
        }
        sl += mm[j] ? l : 0.f;
        sc += (mm[j] && clip) ? 1 : 0;
        g[j] = mm[j] ? d * w : 0.f;
      }
      if (grad != nullptr) {
        if (VEC == 4)
          *reinterpret_cast<float4*>(gp + t) = make_float4(g[0], g[1 % VEC], g[2 % VEC], g[3 % VEC]);
        else
          gp[t] = g[0];
      }
    }
    loss += static_cast<double>(sl) * w;
    kl += sk;
    clipped += sc;
  }
  loss = warp_sum_d(loss);
  kl = warp_sum_d(kl);
  clipped = warp_sum_d(clipped);
  if (lane == 0) {
    s_sum[0][warp] = loss;
    s_sum[1][warp] = kl;
    s_sum[2][warp] = clipped;
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double t = 0.0;
    for (int w = 0; w < 8; ++w) t += s_sum[threadIdx.x][w];
    block_sums[blockIdx.x * 3 + threadIdx.x] = t;
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (s_last && warp < 3) {
    __threadfence();
    double t = 0.0;
    for (int b = lane; b < gridDim.x; b += 32) t += static_cast<volatile double*>(block_sums)[b * 3 + warp];
    t = warp_sum_d(t);
    if (lane == 0) {
      if (warp == 0) *loss_out = static_cast<float>(t);
      else *(warp == 1 ? kl_out : clipped_out) = static_cast<float>(t * inv_tokens);
    }
  }
}

// x *= *s, unless *s is 1 (the usual gradient of a loss): then nothing is read or written and the
// launch costs 2 us
template <int VEC>
__global__ void __launch_bounds__(256) scale_unless_one_kernel(float* __restrict__ x, long long n,
                                                               const float* __restrict__ s) {
  const float c = *s;
  if (c == 1.f) return;
  const long long step = static_cast<long long>(gridDim.x) * 256 * VEC;
  for (long long i = (blockIdx.x * 256LL + threadIdx.x) * VEC; i < n; i += step) {
    if (VEC == 4 && i + 4 <= n) {
      float4 v = *reinterpret_cast<float4*>(x + i);
      v.x *= c; v.y *= c; v.z *= c; v.w *= c;
      *reinterpret_cast<float4*>(x + i) = v;
    } else {
      for (long long j = i; j < min(n, i + VEC); ++j) x[j] *= c;
    }
  }
}

// ------------------------------------------------------------------------ MoE router
// A row of E logits is held by a group of G lanes, NV vectors of VEC per lane (column
// (v G + lane) VEC + j). One row then costs log2(G) shuffle steps shared by 32 / G rows.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC, int NV>
struct RowRaw {
  Pack<T, VEC> v[NV];
};

// a lane's part of one row as stored; p points at the lane's first column. Columns past E (a
// multiple of VEC) are not read: FULL rows have none.
template <typename T, int VEC, int G, int NV, bool FULL>
__device__ __forceinline__ void fetch_row(const T* p, int sub, int E, RowRaw<T, VEC, NV>& x) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (FULL || (v * G + sub) * VEC < E) x.v[v] = *reinterpret_cast<const Pack<T, VEC>*>(p + v * G * VEC);
}

// bf16 values are the upper halves of fp32 ones: one shift or mask each
__device__ __forceinline__ float pair_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float pair_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

template <typename T, int VEC, int G, int NV, bool FULL>
__device__ __forceinline__ void unpack_row(const RowRaw<T, VEC, NV>& r, int sub, int E, float (&x)[NV * VEC]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const bool has = FULL || (v * G + sub) * VEC < E;
    if (sizeof(T) == 2 && VEC == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(&r.v[v]);
      const uint32_t* w = &u.x;
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        x[v * VEC + 2 * j] = has ? pair_lo(w[j]) : -INFINITY;
        x[v * VEC + (2 * j + 1) % VEC] = has ? pair_hi(w[j]) : -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[v * VEC + j] = has ? static_cast<float>(r.v[v].v[j]) : -INFINITY;
    }
  }
}

// Walks a warp's rows through the layers' matrices: kGroups = 32 / G neighbouring rows a step,
// a group of lanes per row, steps of all warps interleaved so that the machine reads one
// window of memory at a time. `p` is the lane's place in its group's current row. Rows number
// fewer than 2^30 (checked by the launcher).
template <typename T, int VEC, int G>
struct RowWalk {
  static constexpr int kGroups = 32 / G;
  const T* p;
  int r, end, t, layer, stride;
  __device__ __forceinline__ RowWalk(const RouterArgs& a, int warp, int warps, int sub, int grp)
      : r(warp * kGroups + grp), end(a.L * static_cast<int>(a.T)), stride(warps * kGroups) {
    layer = r / static_cast<int>(a.T);
    t = r - layer * static_cast<int>(a.T);
    place(a, sub);
  }
  __device__ __forceinline__ void place(const RouterArgs& a, int sub) {
    if (r < end) p = static_cast<const T*>(a.logits[layer]) + t * a.ld[layer] + sub * VEC;
  }
  __device__ __forceinline__ bool in() const { return r < end; }
  // the row's mask byte, fetched beside the row: a row that does not count is read all the
  // same, so that its load does not wait for the byte
  __device__ __forceinline__ uint8_t mask(const RouterArgs& a) const {
    return a.mask == nullptr ? 1 : a.mask[t];
  }
  __device__ __forceinline__ void next(const RouterArgs& a, int sub) {
    const int T_ = static_cast<int>(a.T);
    r += stride;
    if (r >= end) return;
    t += stride;
    while (t >= T_) {
      t -= T_;
      ++layer;
    }
    place(a, sub);
  }
};

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Blocks an SM: the sums keep 32 bf16 values a lane (fewer shuffles and scalar steps for a row:
// 97 us instead of 130 with 16, 24 x 32768 x 256), the gradient 16.
constexpr int kRouterThreads = 256, kRouterSumsResident = 2, kRouterGradResident = 4;

// Per block: column sums of the probabilities, the sum of lse^2, the kept tokens and the
// histogram of the chosen experts over the block's rows; lse of every row for the backward.
// A row lies in the registers of a group of lanes, so its maximum, sum and probabilities take one
// read and no shared memory. Bound by instructions (exponential, sums, shuffles) together with
// memory: 24 x 32768 x 256 bf16 and 8 indices each, 453 MB in 101 us, 4.5 TB/s.
template <typename T, int VEC, int G, int NV, bool FULL>
__global__ void __launch_bounds__(kRouterThreads, kRouterSumsResident) router_sums_kernel(const __grid_constant__ RouterArgs a,
                                                                     float* __restrict__ lse_out,
                                                                     float* __restrict__ part_p,
                                                                     int* __restrict__ part_n,
                                                                     double* __restrict__ part_z,
                                                                     unsigned* __restrict__ ticket) {
  dependents_may_start();
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
  constexpr int kEl = NV * VEC, kCover = G * kEl, kGroups = 32 / G, kWarps = kRouterThreads / 32;
  static_assert(kEl % 2 == 0, "values are processed in pairs");
  __shared__ float s_p[kCover];
  __shared__ int s_hist[kCover];
  __shared__ double s_z[kWarps];
  __shared__ int s_kept[kWarps], s_bad;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (G - 1), grp = lane / G;
  for (int i = threadIdx.x; i < kCover; i += kRouterThreads) {
    s_p[i] = 0.f;
    s_hist[i] = 0;
  }
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  float acc[kEl];
#pragma unroll
  for (int i = 0; i < kEl; ++i) acc[i] = 0.f;
  double z = 0.0;
  int kept = 0;
  // each row is fetched one step ahead
  RowWalk<T, VEC, G> w(a, blockIdx.x * kWarps + warp, gridDim.x * kWarps, sub, grp);
  RowRaw<T, VEC, NV> raw;
  uint8_t keep = 0;
  if (w.in()) {
    keep = w.mask(a);
    fetch_row<T, VEC, G, NV, FULL>(w.p, sub, a.E, raw);
  }
  float zf = 0.f;
  while (__any_sync(0xffffffffu, w.in())) {
    const int r = w.r;
    const bool kept_row = w.in() && keep != 0;
    // the row's chosen experts, spread over its lanes: read here, counted after the arithmetic
    const int64_t* ip = w.in() ? a.idx[w.layer] + static_cast<long long>(w.t) * a.k : nullptr;
    int64_t chosen[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) chosen[j] = w.in() && sub + j * G < a.k ? ip[sub + j * G] : -1;
    float x[kEl];
    unpack_row<T, VEC, G, NV, FULL>(raw, sub, a.E, x);
    w.next(a, sub);
    if (w.in()) {
      keep = w.mask(a);
      fetch_row<T, VEC, G, NV, FULL>(w.p, sub, a.E, raw);
    }
    // exponentials relative to the lane's own maximum, so that they do not wait for the row's
    float ml = fmax3(x[0], x[1], x[2 % kEl]);
#pragma unroll
    for (int e = 3; e + 1 < kEl; e += 2) ml = fmax3(ml, x[e], x[e + 1]);
    ml = fmaxf(ml, x[kEl - 1]) * kLog2e;
    const float off = ml == -INFINITY ? 0.f : ml;  // a lane past the last column
    float s = 0.f, s1 = 0.f;
#pragma unroll
    for (int e = 0; e < kEl; e += 2) {
      ffma2(x[e], x[e + 1], x[e], x[e + 1], kLog2e, kLog2e, -off, -off);
      x[e] = fast_exp2(x[e]);
      x[e + 1] = fast_exp2(x[e + 1]);
      fadd2(s, s1, s, s1, x[e], x[e + 1]);
    }
    const float m = group_max<G>(ml), to_row = fast_exp2(ml - m);
    s = group_sum<G>((s + s1) * to_row);
    const float inv = __fdividef(to_row, s), lse = kLn2 * (m + log2f(s));
    if (kept_row) {
#pragma unroll
      for (int e = 0; e < kEl; e += 2) ffma2(acc[e], acc[e + 1], x[e], x[e + 1], inv, inv, acc[e], acc[e + 1]);
      if (sub == 0) {
        zf = fmaf(lse, lse, zf);
        ++kept;
        lse_out[r] = lse;
      }
      for (int j = sub; j < a.k; j += G) {
        const int64_t e = j < G ? chosen[0] : j < 2 * G ? chosen[1] : ip[j];
        if (e >= 0 && e < a.E) atomicAdd(&s_hist[e], 1);
        else s_bad = 1;
      }
    }
  }
  z = zf;
  // the warps add their column sums in turn: a fixed order
#pragma unroll
  for (int i = 0; i < kEl; ++i) {
#pragma unroll
    for (int o = 16; o >= G; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  }
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp && grp == 0) {
#pragma unroll
      for (int i = 0; i < kEl; ++i) s_p[((i / VEC) * G + sub) * VEC + i % VEC] += acc[i];
    }
    __syncthreads();
  }
  z = warp_sum_d(z);
  kept = __reduce_add_sync(0xffffffffu, kept);
  if (lane == 0) {
    s_z[warp] = z;
    s_kept[warp] = kept;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.E; i += kRouterThreads) {
    part_p[static_cast<long long>(blockIdx.x) * a.E + i] = s_p[i];
    part_n[static_cast<long long>(blockIdx.x) * a.E + i] = s_hist[i];
  }
  if (threadIdx.x == 0) {
    long long n = 0;
    z = 0.0;
    for (int w = 0; w < kWarps; ++w) {
      z += s_z[w];
      n += s_kept[w];
    }
    part_z[blockIdx.x * 2] = z;
    // a NaN marks a chosen index outside [0, E): all fractions, so the loss and the gradient of
    // every kept row, become NaN with it
    part_z[blockIdx.x * 2 + 1] = s_bad ? __longlong_as_double(0x7ff8000000000000LL) : static_cast<double>(n);
  }
}

// Joins the partial sums, 32 columns a block; the last block to finish adds the blocks' parts
// of the loss in their order (9 to 11 us, latency). counts, and the backward's constants
//   slope[e] = c_b E / n * f_e  and  slope[E] = 2 c_z / n
__global__ void __launch_bounds__(1024) router_join_kernel(const float* __restrict__ part_p,
                                                           const int* __restrict__ part_n,
                                                           const double* __restrict__ part_z, int blocks,
                                                           int E, float balance, float zcoef,
                                                           double* __restrict__ dots,
                                                           unsigned* __restrict__ ticket,
                                                           float* __restrict__ loss,
                                                           int64_t* __restrict__ counts,
                                                           float* __restrict__ slope) {
  __shared__ double s_p[32][33];
  __shared__ int s_n[32][33];
  __shared__ double s_tot[2];
  __shared__ bool s_last;
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  double p = 0.0;
  int n = 0;  // at most L T k < 2^31 choices, checked by the launcher
  if (c < E) {
    // every load in flight at once: this kernel is one trip to memory
    constexpr int kTrips = (148 * kRouterSumsResident + 31) / 32;
    float pv[kTrips];
    int nv[kTrips];
#pragma unroll
    for (int i = 0; i < kTrips; ++i) {
      const int b = warp + 32 * i;
      pv[i] = b < blocks ? part_p[static_cast<long long>(b) * E + c] : 0.f;
      nv[i] = b < blocks ? part_n[static_cast<long long>(b) * E + c] : 0;
    }
#pragma unroll
    for (int i = 0; i < kTrips; ++i) {
      p += pv[i];
      n += nv[i];
    }
  }
  s_p[warp][lane] = p;
  s_n[warp][lane] = n;
  if (warp == 1) {
    double z = 0.0, k = 0.0;
    for (int b = lane; b < blocks; b += 32) {
      z += part_z[2 * b];
      k += part_z[2 * b + 1];
    }
    z = warp_sum_d(z);
    k = warp_sum_d(k);
    if (lane == 0) {
      s_tot[0] = z;
      s_tot[1] = k == 0.0 ? 1.0 : k;
    }
  }
  __syncthreads();
  if (warp != 0) return;
  const double tokens = s_tot[1];
  double dot = 0.0;
  if (c < E) {
    long long total = 0;
    p = 0.0;
    for (int w = 0; w < 32; ++w) {
      p += s_p[w][lane];
      total += s_n[w][lane];
    }
    const double f = static_cast<double>(total) / tokens;
    counts[c] = total;
    slope[c] = static_cast<float>(balance * E / tokens * f);
    dot = f * (p / tokens);
  }
  dot = warp_sum_d(dot);
  if (lane == 0) {
    dots[blockIdx.x] = dot;
    __threadfence();
    s_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncwarp();
  if (s_last && lane == 0) {
    __threadfence();
    double t = 0.0;
    for (int b = 0; b < gridDim.x; ++b) t += static_cast<volatile double*>(dots)[b];
    *loss = static_cast<float>(balance * E * t + (zcoef != 0.f ? zcoef * s_tot[0] / tokens : 0.0));
    slope[E] = static_cast<float>(2.0 * zcoef / tokens);
  }
}

// dlogit = gout p (slope_e - <p, slope> + slope_E lse), 0 in masked rows. The probabilities are
// taken from the logits and lse again: half the bytes of storing them. Bound by memory: 24 x 32768
// x 256 bf16 read and written, 805 MB in 128 us, 6.3 TB/s, 0.96 of the measured copy rate (the
// last rows first, so that some are still in L2, gained 0.3%: not kept).
template <typename T, int VEC, int G, int NV, bool FULL>
__global__ void __launch_bounds__(kRouterThreads, NV * VEC > 16 ? 2 : sizeof(T) == 2 ? kRouterGradResident : 3) router_grad_kernel(const __grid_constant__ RouterArgs a,
                                                                     const float* __restrict__ lse_in,
                                                                     const float* __restrict__ slope,
                                                                     const float* __restrict__ gout,
                                                                     T* __restrict__ grad) {
  constexpr int kEl = NV * VEC, kGroups = 32 / G, kWarps = kRouterThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (G - 1), grp = lane / G;
  const float go = *gout, zs = slope[a.E] * go;
  float f[kEl];
#pragma unroll
  for (int i = 0; i < kEl; ++i) {
    const int c = ((i / VEC) * G + sub) * VEC + i % VEC;
    f[i] = c < a.E ? slope[c] * go : 0.f;
  }
  RowWalk<T, VEC, G> w(a, blockIdx.x * kWarps + warp, gridDim.x * kWarps, sub, grp);
  RowRaw<T, VEC, NV> raw;
  float lse_next = 0.f;
  uint8_t keep = 0;
  auto fetch = [&] {
    if (w.in()) {
      keep = w.mask(a);
      lse_next = lse_in[w.r];  // not written for rows that do not count, and not used there
      fetch_row<T, VEC, G, NV, FULL>(w.p, sub, a.E, raw);
    }
  };
  fetch();
  while (__any_sync(0xffffffffu, w.in())) {
    T* g = grad + static_cast<long long>(w.r) * a.E + sub * VEC;
    const bool now = w.in(), kept = now && keep != 0;
    float x[kEl];
    unpack_row<T, VEC, G, NV, FULL>(raw, sub, a.E, x);
    const float lse = lse_next, l2 = lse * kLog2e;
    w.next(a, sub);
    fetch();
    float d = 0.f, d1 = 0.f;
#pragma unroll
    for (int e = 0; e < kEl; e += 2) {
      x[e] = fast_exp2(fmaf(x[e], kLog2e, -l2));
      x[e + 1] = fast_exp2(fmaf(x[e + 1], kLog2e, -l2));
      d = fmaf(x[e], f[e], d);
      d1 = fmaf(x[e + 1], f[e + 1], d1);
    }
    d = group_sum<G>(d + d1);
    const float c = zs * lse - d;
    if (now) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (FULL || (v * G + sub) * VEC < a.E) {
          Pack<T, VEC> u;
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            u.v[j] = static_cast<T>(kept ? x[v * VEC + j] * (f[v * VEC + j] + c) : 0.f);
          *reinterpret_cast<Pack<T, VEC>*>(g + v * G * VEC) = u;
        }
      }
    }
  }
}

int warp_grid(long long units) {
  return static_cast<int>(std::max<long long>(1, std::min<long long>((units + 7) / 8, 148 * 8)));
}

int warp_tokens(long long rows, int S) {
  int len = kMaxWarpTokens;
  while (len > kMinWarpTokens && rows * ((S + len - 1) / len) < 148LL * 16) len /= 2;
  return len;
}

int chunks_of(long long rows, int S) {
  const int len = warp_tokens(rows, S);
  return std::max(1, (S + len - 1) / len);
}

// 4 tokens at a time need every row to start on a boundary of 4 elements
bool aligned4(const void* p, int bytes, std::initializer_list<long long> strides) {
  if (reinterpret_cast<uintptr_t>(p) % (4 * bytes)) return false;
  for (long long s : strides)
    if (s % 4) return false;
  return true;
}

// The layout for E columns: 16-byte vectors where every row allows them, PER_LANE values a lane
// in the fewest lanes that hold a row (twice as many where 32 lanes do not); FULL where they
// hold exactly it.
template <typename T, int PER_LANE, typename F>
void router_dispatch(int E, bool vec, F&& launch) {
  constexpr int V = 16 / sizeof(T), N = PER_LANE / V, K = PER_LANE;
  auto pick = [&](auto VEC, auto G, auto NV) {
    if (E == VEC.value * G.value * NV.value) launch(VEC, G, NV, std::true_type{});
    else launch(VEC, G, NV, std::false_type{});
  };
  using std::integral_constant;
  if (vec) {
    if (E <= K) pick(integral_constant<int, V>{}, integral_constant<int, 1>{}, integral_constant<int, N>{});
    else if (E <= 2 * K) pick(integral_constant<int, V>{}, integral_constant<int, 2>{}, integral_constant<int, N>{});
    else if (E <= 4 * K) pick(integral_constant<int, V>{}, integral_constant<int, 4>{}, integral_constant<int, N>{});
    else if (E <= 8 * K) pick(integral_constant<int, V>{}, integral_constant<int, 8>{}, integral_constant<int, N>{});
    else if (E <= 16 * K) pick(integral_constant<int, V>{}, integral_constant<int, 16>{}, integral_constant<int, N>{});
    else if (E <= 32 * K) pick(integral_constant<int, V>{}, integral_constant<int, 32>{}, integral_constant<int, N>{});
    else if constexpr (K < 32) pick(integral_constant<int, V>{}, integral_constant<int, 32>{}, integral_constant<int, 2 * N>{});
  } else {
    using One = integral_constant<int, 1>;
    using Warp = integral_constant<int, 32>;
    if (E <= 128) launch(One{}, Warp{}, integral_constant<int, 4>{}, std::false_type{});
    else if (E <= 256) launch(One{}, Warp{}, integral_constant<int, 8>{}, std::false_type{});
    else if (E <= 512) launch(One{}, Warp{}, integral_constant<int, 16>{}, std::false_type{});
    else launch(One{}, Warp{}, integral_constant<int, 32>{}, std::false_type{});
  }
}

template <typename T>
bool router_vec(const RouterArgs& a) {
  constexpr int V = 16 / sizeof(T);
  if (a.E % V) return false;
  for (int l = 0; l < a.L; ++l)
    if (a.ld[l] % V || (reinterpret_cast<uintptr_t>(a.logits[l]) & 15)) return false;
  return true;
}

}  // namespace

int pref_chunks(int P, int S) { return chunks_of(2LL * P, S); }

int pref_blocks(int P) { return std::max(1, std::min((P + 7) / 8, 148)); }

void pref_forward(const PrefArgs& a, void* part, double* block_loss, unsigned* ticket, float* row_scale,
                  float* loss, float* chosen, float* rejected, cudaStream_t st) {
  if (a.P <= 0) return;
  const int chunks = pref_chunks(a.P, a.S), len = warp_tokens(2LL * a.P, a.S);
  const bool vec = a.S % 4 == 0 && aligned4(a.logps, 4, {a.lp_side, a.lp_pair}) &&
                   aligned4(a.mask, 1, {a.mk_side, a.mk_pair}) &&
                   (a.ref == nullptr || aligned4(a.ref, a.ref_bf16 ? 2 : 4, {a.ref_side, a.ref_pair}));
  const int grid = warp_grid(2LL * a.P * chunks);
  if (vec) pref_sums_kernel<4><<<grid, 256, 0, st>>>(a, static_cast<float2*>(part), chunks, len, ticket);
  else pref_sums_kernel<1><<<grid, 256, 0, st>>>(a, static_cast<float2*>(part), chunks, len, ticket);
  PLG_CUDA_CHECK(cudaGetLastError());
  launch_dependent(pref_pairs_kernel, pref_blocks(a.P), 256, st, a, static_cast<const float2*>(part), chunks,
                   block_loss, ticket, row_scale, loss, chosen, rejected);
}

void pref_backward(const PrefArgs& a, const float* row_scale, const float* gout, float* grad, cudaStream_t st) {
  if (a.P <= 0 || a.S <= 0) return;
  const int chunks = pref_chunks(a.P, a.S), len = warp_tokens(2LL * a.P, a.S);
  const bool vec = a.S % 4 == 0 && aligned4(a.mask, 1, {a.mk_side, a.mk_pair}) && aligned4(grad, 4, {});
  const int grid = warp_grid(2LL * a.P * chunks);
  if (vec) pref_grad_kernel<4><<<grid, 256, 0, st>>>(a, row_scale, gout, grad, chunks, len);
  else pref_grad_kernel<1><<<grid, 256, 0, st>>>(a, row_scale, gout, grad, chunks, len);
  PLG_CUDA_CHECK(cudaGetLastError());
}

int policy_count_blocks(int R, int S) {
  const long long b = S > 2048 ? R : (R + 7) / 8;
  return static_cast<int>(std::max<long long>(1, std::min<long long>(b, 148 * 4)));
}

// as many blocks as stay resident (registers allow 3 an SM): each warp takes several units
int policy_blocks(int R, int S) {
  return std::min(warp_grid(static_cast<long long>(R) * chunks_of(R, S)), 148 * kPolicyResident);
}

void policy_forward(const PolicyArgs& a, int* counts, void* block_counts, double* block_sums,
                    unsigned* ticket, float* grad, float* loss, float* kl, float* clipped, cudaStream_t st) {
  if (a.R <= 0) return;
  const int cb = policy_count_blocks(a.R, a.S);
  longlong2* bc = static_cast<longlong2*>(block_counts);
  if (a.S > 2048) policy_counts_kernel<true><<<cb, 256, 0, st>>>(a, counts, bc, ticket);
  else policy_counts_kernel<false><<<cb, 256, 0, st>>>(a, counts, bc, ticket);
  PLG_CUDA_CHECK(cudaGetLastError());
  const int chunks = chunks_of(a.R, a.S), len = warp_tokens(a.R, a.S);
  const bool vec = a.S % 4 == 0 && aligned4(a.logps, 4, {a.lp_row}) && aligned4(a.mask, 1, {a.mk_row}) &&
                   (a.old == nullptr || aligned4(a.old, a.old_bf16 ? 2 : 4, {a.old_row})) &&
                   (a.ref == nullptr || aligned4(a.ref, a.ref_bf16 ? 2 : 4, {a.ref_row})) &&
                   (a.adv_tok == 0 || aligned4(a.adv, 4, {a.adv_row})) && aligned4(grad, 4, {});
  const int grid = policy_blocks(a.R, a.S);
  auto launch = [&](auto old, auto ref, auto adv) {
    auto kern = vec ? policy_kernel<4, old.value, ref.value, adv.value>
                    : policy_kernel<1, old.value, ref.value, adv.value>;
    launch_dependent(kern, grid, 256, st, a, counts, bc, cb, block_sums, ticket, grad, loss, kl, clipped, chunks, len);
  };
  auto pick = [&](auto old, auto ref) {
    if (a.adv_tok) launch(old, ref, std::true_type{});
    else launch(old, ref, std::false_type{});
  };
  auto pick_ref = [&](auto old) {
    if (a.ref != nullptr) pick(old, std::true_type{});
    else pick(old, std::false_type{});
  };
  if (a.old != nullptr) pick_ref(std::true_type{});
  else pick_ref(std::false_type{});
  PLG_CUDA_CHECK(cudaGetLastError());
}

void scale_unless_one(float* x, long long n, const float* s, cudaStream_t st) {
  if (n <= 0) return;
  const int grid = static_cast<int>(std::min<long long>((n + 1023) / 1024, 148 * 8));
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) scale_unless_one_kernel<4><<<grid, 256, 0, st>>>(x, n, s);
  else scale_unless_one_kernel<1><<<grid, 256, 0, st>>>(x, n, s);
  PLG_CUDA_CHECK(cudaGetLastError());
}

int router_blocks(long long rows) {
  // at least 64 rows a block
  return static_cast<int>(std::max<long long>(1, std::min<long long>((rows + 63) / 64, 148 * kRouterSumsResident)));
}

void router_balance_forward(const RouterArgs& a, bool bf16, float balance, float zcoef, float* lse,
                            float* part_p, int* part_n, double* part_z, double* dots, unsigned* ticket,
                            float* loss, int64_t* counts, float* slope, cudaStream_t st) {
  if (a.E < 1 || a.E > kRouterMaxExperts || a.L < 1 || a.L > kRouterMaxLayers || a.k < 0)
    throw std::invalid_argument("router_balance_loss: 1..1024 experts and 1..128 layers in one call");
  const long long rows = static_cast<long long>(a.L) * a.T;
  if (rows >= 1 << 30 || rows * std::max(a.k, 1) > INT32_MAX)
    throw std::invalid_argument("router_balance_loss: more than 2^30 rows or 2^31 choices in one call");
  const int blocks = router_blocks(rows);
  if (rows == 0) PLG_CUDA_CHECK(cudaMemsetAsync(ticket, 0, sizeof(unsigned), st));
  if (rows > 0) {
    auto run = [&](auto* tag, bool vec) {
      using T = std::remove_pointer_t<decltype(tag)>;
      router_dispatch<T, sizeof(T) == 2 ? 32 : 16>(a.E, vec, [&](auto V, auto G, auto N, auto FULL) {
        router_sums_kernel<T, V.value, G.value, N.value, FULL.value><<<blocks, kRouterThreads, 0, st>>>(a, lse, part_p, part_n,
                                                                                          part_z, ticket);
      });
    };
    if (bf16) run(static_cast<__nv_bfloat16*>(nullptr), router_vec<__nv_bfloat16>(a));
    else run(static_cast<float*>(nullptr), router_vec<float>(a));
    PLG_CUDA_CHECK(cudaGetLastError());
  }
  launch_dependent(router_join_kernel, (a.E + 31) / 32, 1024, st, part_p, part_n, part_z, rows > 0 ? blocks : 0, a.E,
                   balance, zcoef, dots, ticket, loss, counts, slope);
}

void router_balance_backward(const RouterArgs& a, bool bf16, const float* lse, const float* slope,
                             const float* gout, void* grad, cudaStream_t st) {
  const long long rows = static_cast<long long>(a.L) * a.T;
  if (rows <= 0) return;
  const int blocks =
      static_cast<int>(std::max<long long>(1, std::min<long long>((rows + 31) / 32, 148 * kRouterGradResident)));
  auto run = [&](auto* tag, bool vec) {
    using T = std::remove_pointer_t<decltype(tag)>;
    vec = vec && (reinterpret_cast<uintptr_t>(grad) & 15) == 0;
    router_dispatch<T, 16>(a.E, vec, [&](auto V, auto G, auto N, auto FULL) {
      router_grad_kernel<T, V.value, G.value, N.value, FULL.value><<<blocks, kRouterThreads, 0, st>>>(a, lse, slope, gout,
                                                                                        static_cast<T*>(grad));
    });
  };
  if (bf16) run(static_cast<__nv_bfloat16*>(nullptr), router_vec<__nv_bfloat16>(a));
  else run(static_cast<float*>(nullptr), router_vec<float>(a));
  PLG_CUDA_CHECK(cudaGetLastError());
}

}  // namespace plg
