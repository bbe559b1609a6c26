// Distillation of the head from a teacher's top logits (no counterpart in the reference).  With the scores
// z = s / tau h W^T + b / tau and their log-sum-exp LSE over the vocabulary, and the teacher's distribution
// p_n = softmax(t_n / tau) over the T entries (id, t) it gives for token n,
//
//   kl[n]   = sum_k p[n,k] (log p[n,k] - z[n, id[n,k]] + LSE[n])
//   loss    = sum_n w[n] (kl[n] + zw LSE[n]^2) * c,     c = 1 / sum_n w[n] (mean), 1 (sum)
//   dS[n,v] = c_n softmax(z)[n,v] - sum over k with id[n,k] = v of g_n p[n,k],
//             g_n = g c w[n],  c_n = g_n (1 + 2 zw LSE[n]);
//   gh = s / tau dS W,   gW = s / tau dS^T h,   gb = colsum(dS) / tau.
//
// LSE and the dense part of the gradients are the readout's forward and backward (with no embedding: D = 0,
// gO = 0, gLSE = c_n), so the [N, V] scores are not in memory but where few tokens' are kept from the forward for the
// backward (fwd_kept_scores).  What is here is the sparse part:
//   distill_dot_kernel    z at the teacher's ids: dot products of h's row with gathered rows of W in fp32
//                         (2 N T K flops; bound by the gather, N T rows of W);
//   distill_loss_kernel   p, the loss's terms and softmax(z) at the ids (one wave per token);
//   distill_prep_kernel   c_n, and the values of dS at the ids, in fp32 and with p taken off there: after the
//                         scores kernel has staged a chunk of dS, bwd_patch_kernel (bwd.hip) writes them over
//                         its elements, so the difference is rounded once, not its two terms;
//   distill_bias_kernel   takes the sums of g_n p off gb, over the entries sorted by id (sort_ids).
// An entry with a negative id or a logit of -inf is absent; a token without entries, or of weight zero, has
// loss 0, no share in c and no gradient.  An id of V or more makes its token's loss NaN, and so are the gradients of
// a token whose divergence is NaN for any reason: coef carries it to them, so that a check of them finds it.
#include <cfloat>

#include "common.hpp"
#include "launch.hpp"

namespace swvr {

namespace {

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

__device__ __forceinline__ int64_t id_at(const DistillParams& p, int n, int k) {
  const int64_t i = (int64_t)n * p.ldi + k;
  return p.id64 ? static_cast<const int64_t*>(p.ids)[i] : (int64_t)static_cast<const int*>(p.ids)[i];
}

__device__ __forceinline__ float load_as(const void* x, int64_t i, int dtype) {
  return dtype == kBF16  ? (float)static_cast<const bf16_t*>(x)[i]
         : dtype == kF16 ? (float)static_cast<const f16_t*>(x)[i]
                         : static_cast<const float*>(x)[i];
}

__global__ __launch_bounds__(256) void distill_scale_kernel(const void* __restrict__ x, int dtype, int64_t n, float s,
                                                            float* __restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) y[i] = load_as(x, i, dtype) * s;
}

// 8 consecutive values of a row stored as S, rounded to the compute dtype T.
template <class T, class S>
__device__ __forceinline__ void load8(const S* row, float (&v)[8]) {
  typedef typename Vec8<S>::type V8;
  const V8 x = *reinterpret_cast<const V8*>(row);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)(T)x[i];
}

// z of IDS entries of a token per wave: h's 8 values of a lane serve them all.  4 where that leaves kManyWaves waves
// (with the whole forward, bf16: 4096 tokens, T = 64, K = 256 111 -> 79 us, K = 4096 436 -> 345; 512 tokens, T = 32,
// K = 4096 83 -> 77); 1 with 4 steps of its row in flight where they are few and each waits for its rows (8 tokens,
// T = 10, K = 4096: 24 -> 6 us; 500, T = 16, K = 4096, with the forward 74.7 -> 71.8).
template <class T, class HS, class WS, int IDS, int STEPS>
__global__ __launch_bounds__(256) void distill_dot_kernel(DistillParams p, int64_t b0) {
  const int groups = (p.T + IDS - 1) / IDS;
  const int64_t gw = (b0 + blockIdx.x) * 4 + wave_id();
  if (gw >= (int64_t)p.N * groups) return;
  const int n = (int)(gw / groups), k0 = (int)(gw % groups) * IDS;
  if (p.weight && p.weight[n] == 0.f) return;
  const int lane = lane_id();
  const HS* const h = static_cast<const HS*>(p.h) + (int64_t)n * p.ldh;
  const WS* w[IDS];
  bool in[IDS];
  int id[IDS];
  bool any = false;
#pragma unroll
  for (int u = 0; u < IDS; ++u) {
    const int64_t x = k0 + u < p.T ? id_at(p, n, k0 + u) : -1;
    in[u] = x >= 0 && x < p.V;
    id[u] = in[u] ? (int)x : 0;
    w[u] = static_cast<const WS*>(p.W) + (int64_t)id[u] * p.ldw;
    any |= in[u];
  }
  if (!any) return;
  float acc[IDS];
#pragma unroll
  for (int u = 0; u < IDS; ++u) acc[u] = 0.f;
  for (int k = lane * 8; k < p.K; k += 512 * STEPS) {
    float a[STEPS][8], b[STEPS][IDS][8];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int at = k + 512 * s < p.K ? k + 512 * s : k;  // (past the row: again, and not added)
      load8<T, HS>(h + at, a[s]);
#pragma unroll
      for (int u = 0; u < IDS; ++u)
        if (in[u]) load8<T, WS>(w[u] + at, b[s][u]);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (k + 512 * s < p.K)
#pragma unroll
        for (int u = 0; u < IDS; ++u)
          if (in[u])
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[u] = fmaf(a[s][i], b[s][u][i], acc[u]);
  }
#pragma unroll
  for (int u = 0; u < IDS; ++u) {
    const float s = wave_sum(acc[u]);
    if (lane == u && in[u]) p.z[(int64_t)n * p.T + k0 + u] = s * p.scale + (p.bias ? p.bias[id[u]] : 0.f);
  }
}

// One wave per token, 4 tokens per workgroup, the workgroup's sums of the terms and of the weights in token order.  The
// first 64 entries stay in registers; longer lists are read again for each of the three passes (the largest, the sum of
// exponentials, the terms).  (4 tokens per wave, one after another, took 11 us for 500 tokens.)
constexpr int kTokensPerBlock = 4;
__global__ __launch_bounds__(256) void distill_loss_kernel(DistillParams p, float* __restrict__ part, int n_blk) {
  __shared__ float s_loss[4], s_w[4];
  const int lane = lane_id(), wv = wave_id();
  const int n = blockIdx.x * kTokensPerBlock + wv;
  float tok = 0.f, w = 0.f;
  if (n < p.N) {
    struct Entry {
      int64_t id;
      float t;  // -inf: absent
    };
    auto entry = [&](int k) {
      Entry e;
      e.id = id_at(p, n, k);
      const float t = load_as(p.teacher, (int64_t)n * p.ldt + k, p.t_dtype);
      e.t = e.id < 0 ? kNegInf : t;
      return e;
    };
    const Entry none{-1, kNegInf};
    const Entry mine = lane < p.T ? entry(lane) : none;
    const float z0 = lane < p.T && mine.id >= 0 && mine.id < p.V ? p.z[(int64_t)n * p.T + lane] : 0.f;
    const float lse = p.lse[n];
    w = p.weight ? p.weight[n] : 1.f;
    // fmaxf leaves a NaN out; it comes back with the exponentials
    float m = mine.t;
    bool has = mine.t != kNegInf;
    for (int k = lane + 64; k < p.T; k += 64) {
      const Entry e = entry(k);
      has |= e.t != kNegInf;
      m = fmaxf(m, e.t);
    }
    m = wave_max(m);
    if (w == 0.f || __ballot(has) == 0) w = 0.f;
    float coef = w;
    if (w != 0.f) {
      // (the distance from the largest before the division: a logit of the type's lowest value stays one at any
      // temperature, where the quotient would be -inf, an absent entry's)
      auto below = [&](float t) { return (t - m) * p.inv_tau; };
      auto mass = [&](float t) { return t != kNegInf ? expf(below(t)) : 0.f; };
      float sum = mass(mine.t);
      for (int k = lane + 64; k < p.T; k += 64) sum += mass(entry(k).t);
      const float lp = logf(wave_sum(sum));
      float kl = 0.f;
      auto term = [&](const Entry& e, int k, float z) {
        const float logq = e.id >= p.V ? __builtin_nanf("") : e.id >= 0 ? z - lse : kNegInf;
        const float logp = below(e.t) - lp, pk = e.t != kNegInf ? expf(logp) : 0.f;
        // (NaN != 0; an id outside the vocabulary shows whatever its probability rounds to)
        if (pk != 0.f || (e.t != kNegInf && e.id >= p.V)) kl += pk * (logp - logq);
        if (p.p) {
          p.p[(int64_t)n * p.T + k] = pk;
          p.q[(int64_t)n * p.T + k] = e.id >= p.V ? 0.f : expf(logq);
        }
      };
      if (lane < p.T) term(mine, lane, z0);
      for (int k = lane + 64; k < p.T; k += 64) {
        const Entry e = entry(k);
        term(e, k, e.id >= 0 && e.id < p.V ? p.z[(int64_t)n * p.T + k] : 0.f);
      }
      tok = wave_sum(kl);
      if (tok != tok) coef = tok;  // the gradients that the token reaches are NaN too
      if (p.zw != 0.f) tok += p.zw * (lse * lse);
      tok *= w;
    } else if (p.p) {
      for (int k = lane; k < p.T; k += 64) p.p[(int64_t)n * p.T + k] = p.q[(int64_t)n * p.T + k] = 0.f;
    }
    if (lane == 0) {
      if (p.coef) p.coef[n] = coef;
      if (p.reduce == 0) p.out[n] = tok;
    }
  }
  if (!part) return;
  if (lane == 0) {
    s_loss[wv] = tok;
    s_w[wv] = w;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    part[blockIdx.x] = ((s_loss[0] + s_loss[1]) + s_loss[2]) + s_loss[3];
    part[n_blk + blockIdx.x] = ((s_w[0] + s_w[1]) + s_w[2]) + s_w[3];
  }
}

// The loss and c from the workgroups' sums; weights that sum to zero leave c = 1 (no token to learn from: 0).
__global__ __launch_bounds__(256) void distill_reduce_kernel(const float* __restrict__ part, int n_blk, int mean,
                                                             float* __restrict__ out, float* __restrict__ c) {
  __shared__ float s_loss[256], s_w[256];
  float a = 0.f, b = 0.f;
  for (int i = threadIdx.x; i < n_blk; i += 256) {
    a += part[i];
    b += part[n_blk + i];
  }
  s_loss[threadIdx.x] = a;
  s_w[threadIdx.x] = b;
  __syncthreads();
  for (int s = 128; s > 0; s >>= 1) {
    if ((int)threadIdx.x < s) {
      s_loss[threadIdx.x] += s_loss[threadIdx.x + s];
      s_w[threadIdx.x] += s_w[threadIdx.x + s];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float denom = mean && s_w[0] != 0.f ? s_w[0] : 1.f;
    out[0] = s_loss[0] / denom;
    c[0] = 1.f / denom;
  }
}

// One wave per token: what the backward's first kernel would make of O = gO = 0 and gLSE = c_n (delta = -c_n and the
// flag of an active token), and per entry the id (-1: no element of its own), dS there, and g_n p.  Entries of a
// token that repeat an id share one element of dS: the first of them holds their sum.  The entries are compared 64
// against 64, one side from a lane's registers at a time.
__global__ __launch_bounds__(256) void distill_prep_kernel(DistillGradParams p) {
  const int n = blockIdx.x * 4 + wave_id();
  if (n >= p.N) return;
  const int lane = lane_id();
  const float w = p.coef[n], g = w == 0.f ? 0.f : p.g[p.reduce == 0 ? n : 0];
  // a cotangent of zero drops the token, as a weight of zero does, whatever it holds
  const float gn = g == 0.f ? 0.f : g * w * (p.reduce == 0 ? 1.f : p.c[0]);
  float cn = p.zw != 0.f && w != 0.f ? gn * (1.f + 2.f * p.zw * p.lse[n]) : gn;
  // the backward leaves out tokens of gLSE = 0: one whose two terms cancel stays
  if (cn == 0.f && gn != 0.f) cn = FLT_MIN;
  if (lane == 0) {
    p.delta[n] = -cn;
    p.flag[n] = cn != 0.f;  // NaN != 0
  }
  // ids as the matrix has them, -1 outside it; a dropped token has none, whatever its p holds
  auto id_of = [&](int k) -> int {
    if (k >= p.T || gn == 0.f) return -1;
    const int64_t i = (int64_t)n * p.ldi + k;
    const int64_t id = p.id64 ? static_cast<const int64_t*>(p.ids)[i] : (int64_t)static_cast<const int*>(p.ids)[i];
    return id >= 0 && id < p.V ? (int)id : -1;
  };
  for (int k = lane; k < (p.T + 63) / 64 * 64; k += 64) {
    const int64_t e = (int64_t)n * p.T + k;
    const int id = id_of(k);
    const float q = k < p.T ? p.q[e] : 0.f;
    bool own = id >= 0;
    float sum = 0.f;
    for (int j0 = 0; j0 < p.T; j0 += 64) {
      const int id_j = j0 == k - lane ? id : id_of(j0 + lane);
      const float p_j = j0 + lane < p.T ? p.p[(int64_t)n * p.T + j0 + lane] : 0.f;
      const int most = min(64, p.T - j0);
      for (int j = 0; j < most; ++j) {
        const bool same = __builtin_amdgcn_readlane(id_j, j) == id;
        own = own && !(same && j0 + j < k);
        sum += same ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p_j), j)) : 0.f;
      }
    }
    if (k < p.T) {
      const float t = gn * sum;
      p.pt_id[e] = own ? id : -1;
      p.pt_val[e] = cn * q - t;
      if (p.pt_t) p.pt_t[e] = t;
    }
  }
}

// gb[v] = (dense[v] - sum of t over the entries of v) / tau in gb's dtype.  A thread per id, and for an id of more
// than kBiasAlone entries a wave.  (A wave for every id, most of which have no entry: 38 us for V = 252561.)
constexpr int kBiasAlone = 4;
__global__ __launch_bounds__(256) void distill_bias_kernel(const int* __restrict__ order, const int* __restrict__ seg,
                                                           const float* __restrict__ t,
                                                           const float* __restrict__ dense, int V, float inv_tau,
                                                           void* __restrict__ gb, int gb_dtype) {
  __shared__ int s_long[256], s_n;
  const int v = blockIdx.x * 256 + threadIdx.x, lane = lane_id();
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  auto store = [&](int at, float sum) {
    const float y = (dense[at] - sum) * inv_tau;
    if (gb_dtype == kBF16)
      static_cast<bf16_t*>(gb)[at] = (bf16_t)y;
    else if (gb_dtype == kF16)
      static_cast<f16_t*>(gb)[at] = (f16_t)y;
    else
      static_cast<float*>(gb)[at] = y;
  };
  if (v < V) {
    const int i0 = seg[v], i1 = seg[v + 1];
    if (i1 - i0 > kBiasAlone) {
      s_long[atomicAdd(&s_n, 1)] = v;  // whose wave takes an id does not matter
    } else {
      float x[kBiasAlone];
#pragma unroll
      for (int u = 0; u < kBiasAlone; ++u) x[u] = i0 + u < i1 ? t[order[i0 + u]] : 0.f;
      store(v, (x[0] + x[1]) + (x[2] + x[3]));
    }
  }
  __syncthreads();
  for (int j = wave_id(); j < s_n; j += 4) {
    const int at = s_long[j], i1 = seg[at + 1];
    float s = 0.f;
    for (int i = seg[at] + lane; i < i1; i += 256) {
      float x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = i + 64 * u < i1 ? t[order[i + 64 * u]] : 0.f;
      s += (x[0] + x[1]) + (x[2] + x[3]);
    }
    s = wave_sum(s);
    if (lane == 0) store(at, s);
  }
}

template <class T, class HS, class WS>
hipError_t dot_launch(const DistillParams& p, hipStream_t stream) {
  constexpr int64_t kManyWaves = 4096;
  const int64_t many = (int64_t)p.N * ((p.T + 3) / 4), few = (int64_t)p.N * p.T;
  return launch_in_parts(((many >= kManyWaves ? many : few) + 3) / 4, 256, [&](int64_t b0, unsigned n) {
    if (many >= kManyWaves)
      distill_dot_kernel<T, HS, WS, 4, 1><<<n, 256, 0, stream>>>(p, b0);
    else
      distill_dot_kernel<T, HS, WS, 1, 4><<<n, 256, 0, stream>>>(p, b0);
  });
}

template <class T>
hipError_t dot_typed(const DistillParams& p, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.h_f32) return p.w_f32 ? dot_launch<T, float, float>(p, stream) : dot_launch<T, float, T>(p, stream);
    if (p.w_f32) return dot_launch<T, T, float>(p, stream);
  }
  return dot_launch<T, T, T>(p, stream);
}

}  // namespace

size_t distill_part_bytes(int64_t N) {
  return (size_t)((N + kTokensPerBlock - 1) / kTokensPerBlock) * 2 * sizeof(float);
}

hipError_t distill_scale(const void* x, int dtype, int64_t n, float s, float* y, hipStream_t stream) {
  if (n == 0) return hipSuccess;
  distill_scale_kernel<<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(x, dtype, n, s, y);
  return hipGetLastError();
}

hipError_t distill_loss(int dtype, const DistillParams& p, float* part, float* c, hipStream_t stream) {
  const int n_blk = (p.N + kTokensPerBlock - 1) / kTokensPerBlock;
  timing_begin(kKindDistill, stream);
  hipError_t e = hipSuccess;
  if (p.N > 0 && p.T > 0) {
    e = dtype == kBF16 ? dot_typed<bf16_t>(p, stream) : dtype == kF16 ? dot_typed<f16_t>(p, stream)
                                                                      : dot_typed<float>(p, stream);
  }
  if (e == hipSuccess && p.N > 0) {
    distill_loss_kernel<<<n_blk, 256, 0, stream>>>(p, p.reduce ? part : nullptr, n_blk);
    e = hipGetLastError();
  }
  if (e == hipSuccess && p.reduce) {
    distill_reduce_kernel<<<1, 256, 0, stream>>>(part, n_blk, p.reduce == 2, p.out, c);
    e = hipGetLastError();
  }
  timing_end(kKindDistill, stream);
  return e;
}

hipError_t distill_prep(const DistillGradParams& p, hipStream_t stream) {
  timing_begin(kKindDistill, stream);
  distill_prep_kernel<<<(unsigned)((p.N + 3) / 4), 256, 0, stream>>>(p);
  timing_end(kKindDistill, stream);
  return hipGetLastError();
}

hipError_t distill_bias(const int* order, const int* seg, const float* t, const float* dense, int V, float inv_tau,
                        void* gb, int gb_dtype, hipStream_t stream) {
  timing_begin(kKindDistill, stream);
  distill_bias_kernel<<<(unsigned)((V + 255) / 256), 256, 0, stream>>>(order, seg, t, dense, V, inv_tau, gb, gb_dtype);
  timing_end(kKindDistill, stream);
  return hipGetLastError();
}

}  // namespace swvr
