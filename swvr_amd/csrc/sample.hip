// One token per row of logits from a given uniform number, under a temperature, top-k, top-p and min-p (no
// counterpart in the reference, whose generation feeds the readout back).
//
// A row's tokens are ordered by logit, the larger first, equal ones by index.  With m the largest logit and
// w_i = exp((l_i - m) / tau), the kept set is a prefix of that order:
//   top-k   its first k tokens;
//   top-p   of those, with sum Z_k, the tokens before which the sum of w is below p Z_k;
//   min-p   w_i >= min_p (w is relative to the largest already).
// The token drawn is the first in index order whose running sum of kept w exceeds u Z, Z the kept tokens' sum.
// NaN counts as -inf (never drawn); a row of nothing else gives token -1.  tau = 0 takes the first token.
//
// Where u Z falls between two running sums decides the token, so sums must not depend on how the row is split
// nor lose small terms: w is computed in fp64 and held as a whole number of 2^-shift (shift = 62 - bits of V, 44 for
// 151936 tokens), whose sums are exact in 64-bit integers in any order, atomics included.  A token whose w rounds to
// 0 (below 2^-45 of the largest) is never drawn.  The logarithm of the drawn token's probability comes from the
// fp64 exponent, not from the rounded w.
#include <cfloat>

#include "common.hpp"
#include "launch.hpp"

namespace swvr {

namespace {

typedef unsigned long long u64;

constexpr int kRowThreads = 1024, kRowWaves = kRowThreads / 64;
constexpr int kLoad = 4;                           // consecutive logits of a thread per step
constexpr int kTile = kRowThreads * kLoad;         // logits of a workgroup's step
constexpr int kBins = 2048;                        // histogram of 11 key bits

// Order-preserving key of a logit: 0 for NaN and -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > kNegInf)) return 0;
  x += 0.f;  // -0 is 0
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  if (key == 0) return kNegInf;
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Logits i0 .. i0 + 3 of a row as keys (0 outside 0 .. V - 1), in one load.  A row may begin anywhere: i0 + lead is
// a multiple of 4, lead the row's distance from a border of 4 elements.
template <class T>
__device__ __forceinline__ void load_keys(const T* row, int64_t i0, int64_t V, uint32_t (&key)[kLoad]) {
  if (i0 >= 0 && i0 + kLoad <= V) {
    struct alignas(kLoad * sizeof(T)) X {
      T v[kLoad];
    };
    const X x = *reinterpret_cast<const X*>(row + i0);
#pragma unroll
    for (int u = 0; u < kLoad; ++u) key[u] = key_of((float)x.v[u]);
  } else {
#pragma unroll
    for (int u = 0; u < kLoad; ++u) key[u] = i0 + u >= 0 && i0 + u < V ? key_of((float)row[i0 + u]) : 0;
  }
}

// 2^t for t <= 0 (0 below -1000): 2^k times the Taylor series of e^(f ln 2), f = t - k in [-1/2, 1/2], to the
// 11th power of f, whose remainder is (ln 2 / 2)^12 / 12! = 7e-15.  t itself is rounded by 7e-15 at t = -45.
__device__ __forceinline__ double exp2_neg(double t) {
  const double k = rint(t), f = t - k;
  double x = 4.4455382718708116e-10;
  x = fma(x, f, 7.054911620801123e-09);
  x = fma(x, f, 1.01780860092397e-07);
  x = fma(x, f, 1.321548679014431e-06);
  x = fma(x, f, 1.5252733804059841e-05);
  x = fma(x, f, 0.0001540353039338161);
  x = fma(x, f, 0.0013333558146428443);
  x = fma(x, f, 0.009618129107628477);
  x = fma(x, f, 0.05550410866482158);
  x = fma(x, f, 0.24022650695910072);
  x = fma(x, f, 0.6931471805599453);
  x = fma(x, f, 1.0);
  return t > -1000 ? ldexp(x, (int)k) : 0.0;
}

// Weights of a row: w = 2^((l - m) to_log2), to_log2 = log2(e) / tau, in fp64.
struct Weigh {
  double m, to_log2, one;  // one: 2^shift
  uint32_t key_m;
  __device__ __forceinline__ double rel(uint32_t key) const {
    const double t = ((double)logit_of(key) - m) * to_log2;
    // (t is NaN where the largest logit is infinite: tokens equal to it, or under an infinite tau)
    return key == key_m ? 1.0 : key != 0 && t <= 0 ? exp2_neg(t) : 0.0;
  }
  // w in units of 2^-shift, to nearest: below 2^52, so the sum's low bits are the whole number
  __device__ __forceinline__ u64 fix(double w) const {
    return (u64)__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ u64 shfl_up64(u64 x, int o) { return __shfl_up(x, o); }
__device__ __forceinline__ u64 wave_sum64(u64 x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Sum over the workgroup, in every thread; s: kRowWaves words of LDS, free again at the next barrier after.
__device__ __forceinline__ u64 block_sum64(u64 x, u64* s) {
  x = wave_sum64(x);
  __syncthreads();
  if (lane_id() == 0) s[wave_id()] = x;
  __syncthreads();
  x = 0;
#pragma unroll 4
  for (int j = 0; j < kRowWaves; ++j) x += s[j];
  return x;
}

// Sum of the threads before this one, and of all (total).
__device__ __forceinline__ u64 block_before64(u64 x, u64* s, u64* total) {
  u64 y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 z = shfl_up64(y, o);
    if (lane_id() >= o) y += z;
  }
  __syncthreads();
  if (lane_id() == 63) s[wave_id()] = y;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll 4
  for (int j = 0; j < kRowWaves; ++j) {
    before += j < wave_id() ? s[j] : 0;
    all += s[j];
  }
  *total = all;
  return before + y - x;
}

// A place in a row's order: tokens (key, index) with a larger key, or the same one and an index up to this.
struct Cut {
  uint32_t key;
  int64_t idx;
  __device__ __forceinline__ bool keeps(uint32_t k, int64_t i) const { return k > key || (k == key && i <= idx); }
};

// A row's settings.
struct RowSettings {
  double tau, p, min_p, u;
  int64_t k;
};
__device__ __forceinline__ RowSettings settings_of(const SampleParams& a, int64_t r) {
  RowSettings s;
  s.tau = a.tau_rows ? (double)a.tau_rows[r] : a.tau;
  s.k = a.k_rows ? (int64_t)a.k_rows[r] : a.k;
  s.p = a.p_rows ? (double)a.p_rows[r] : a.p;
  s.min_p = a.min_p_rows ? (double)a.min_p_rows[r] : a.min_p;
  s.u = a.u64 ? static_cast<const double*>(a.u)[r] : (double)static_cast<const float*>(a.u)[r];
  if (s.k <= 0 || s.k > a.V) s.k = a.V;
  if (!(s.u >= 0)) s.u = 0;
  if (!(s.tau > 0)) s.tau = 0;
  if (!(s.min_p > 0)) s.min_p = 0;
  return s;
}

// ---------------------------------------------------------------- a row by one workgroup
// Passes over the row: the maximum; for top-k and top-p each, the cut by radix descent over the 32 key bits (11, 11
// and 10 bits: a histogram of counts and weights, the bin where the count reaches k or the weight p Z_k), then the
// place of the last kept one among equal logits; the kept sum; and the running sum up to the token.
template <class T>
struct RowSampler {
  const T* row;
  int64_t V;
  int lead;  // the row's distance from a load border, in elements
  Weigh wt;
  u64* s_sum;        // [kRowWaves]
  uint32_t* s_cnt;   // [kBins]
  u64* s_w;          // [kBins]
  u64* s_out;        // [4]

  template <class F>
  __device__ __forceinline__ void each(F&& f) {  // f(first index, keys), tiles in index order
#pragma unroll 1
    for (int64_t t0 = -lead; t0 < V; t0 += kTile) {
      const int64_t i0 = t0 + threadIdx.x * kLoad;
      uint32_t key[kLoad];
      load_keys(row, i0, V, key);
      f(i0, key);
    }
  }

  // The prefix of the order given by `limit` tokens (by_weight false) or by the tokens before which the
  // weight is below `limit` (by_weight); the weight of the prefix in *sum.
  __device__ Cut select(bool by_weight, double limit, u64* sum) {
    uint32_t lo = 0, hi = 0xffffffffu;
    u64 above_w = 0, above_n = 0, ties = 0;
#pragma unroll 1
    for (;;) {
      const uint32_t span = hi - lo;
      const int bits = span == 0 ? 0 : 32 - __clz(span);
      const int sh = bits > 11 ? bits - 11 : 0;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += kRowThreads) {
        s_cnt[i] = 0;
        s_w[i] = 0;
      }
      __syncthreads();
      each([&](int64_t i0, const uint32_t(&key)[kLoad]) {
#pragma unroll
        for (int u = 0; u < kLoad; ++u) {
          if (key[u] == 0 || key[u] < lo || key[u] > hi) continue;
          const int b = (int)((key[u] - lo) >> sh);
          atomicAdd(&s_cnt[b], 1u);
          const u64 w = wt.fix(wt.rel(key[u]));
          if (w) atomicAdd(&s_w[b], w);
        }
      });
      __syncthreads();
      // from the top bin down: thread t takes bins kBins - 1 - 2t and the one below
      const int b1 = kBins - 1 - 2 * (int)threadIdx.x, b0 = b1 - 1;
      const u64 w1 = s_w[b1], w0 = s_w[b0], n1 = s_cnt[b1], n0 = s_cnt[b0];
      u64 all_w, all_n;
      const u64 bw = above_w + block_before64(w1 + w0, s_sum, &all_w);
      const u64 bn = above_n + block_before64(n1 + n0, s_sum, &all_n);
      if (threadIdx.x == 0) s_out[0] = ~0ull;
      __syncthreads();
      auto hit = [&](int b, u64 w, u64 n, u64 w_before, u64 n_before) {
        // the last bin that begins inside the prefix and holds a token
        const bool in = n > 0 && (by_weight ? (double)w_before < limit : (double)n_before < limit);
        const bool last = by_weight ? (double)(w_before + w) >= limit : (double)(n_before + n) >= limit;
        if (in && last) {
          s_out[0] = b;
          s_out[1] = w_before;
          s_out[2] = n_before;
          s_out[3] = n;
        }
      };
      hit(b1, w1, n1, bw, bn);
      hit(b0, w0, n0, bw + w1, bn + n1);
      __syncthreads();
      const u64 b = s_out[0];
      if (b == ~0ull) {  // the prefix takes every token
        *sum = above_w + all_w;
        return Cut{0, -1};
      }
      above_w = s_out[1];
      above_n = s_out[2];
      ties = s_out[3];
      lo = lo + ((uint32_t)b << sh);
      const uint32_t end = lo + (sh ? (1u << sh) - 1 : 0u);
      hi = end < hi ? end : hi;
      if (lo == hi) break;
    }
    // tokens of key lo, `ties` of them after above_n: how many the prefix takes
    const u64 w = wt.fix(wt.rel(lo));
    u64 take = ties;
    if (by_weight) {
      if (w > 0) {
        const double x = ceil((limit - (double)above_w) / (double)w);
        take = x < 1 ? 1 : x < (double)ties ? (u64)x : ties;
      }
    } else {
      take = (u64)limit - above_n;
    }
    *sum = above_w + take * w;
    if (take >= ties) return Cut{lo, V};
    // the take-th of them in index order
    u64 seen = 0;
    __syncthreads();  // s_out has been read
    if (threadIdx.x == 0) s_out[0] = 0;
#pragma unroll 1
    for (int64_t t0 = -lead; t0 < V && seen < take; t0 += kTile) {
      const int64_t i0 = t0 + threadIdx.x * kLoad;
      uint32_t key[kLoad];
      load_keys(row, i0, V, key);
      u64 n = 0;
#pragma unroll
      for (int u = 0; u < kLoad; ++u) n += key[u] == lo;
      u64 all;
      u64 at = seen + block_before64(n, s_sum, &all);
#pragma unroll
      for (int u = 0; u < kLoad; ++u)
        if (key[u] == lo && ++at == take) s_out[0] = (u64)(i0 + u);
      seen += all;
    }
    __syncthreads();
    return Cut{lo, (int64_t)s_out[0]};
  }
};

template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleParams a) {
  __shared__ u64 s_sum[kRowWaves], s_w[kBins], s_out[4];
  __shared__ uint32_t s_cnt[kBins];
  __shared__ uint32_t s_key[kRowWaves];
  __shared__ int64_t s_idx[kRowWaves];
  const int64_t r = blockIdx.x;
  const RowSettings s = settings_of(a, r);
  RowSampler<T> q;
  q.row = static_cast<const T*>(a.logits) + r * a.ld;
  q.V = a.V;
  q.lead = (int)((reinterpret_cast<uintptr_t>(q.row) / sizeof(T)) % kLoad);
  q.s_sum = s_sum;
  q.s_w = s_w;
  q.s_cnt = s_cnt;
  q.s_out = s_out;
  // the largest logit, the first of equal ones
  uint32_t km = 0;
  int64_t im = a.V;
  q.each([&](int64_t i0, const uint32_t(&key)[kLoad]) {
#pragma unroll
    for (int u = 0; u < kLoad; ++u)
      if (key[u] > km) {
        km = key[u];
        im = i0 + u;
      }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t k2 = __shfl_xor(km, o);
    const int64_t i2 = __shfl_xor(im, o);
    if (k2 > km || (k2 == km && i2 < im)) {
      km = k2;
      im = i2;
    }
  }
  if (lane_id() == 0) {
    s_key[wave_id()] = km;
    s_idx[wave_id()] = im;
  }
  __syncthreads();
  for (int j = 0; j < kRowWaves; ++j)
    if (s_key[j] > km || (s_key[j] == km && s_idx[j] < im)) {
      km = s_key[j];
      im = s_idx[j];
    }
  if (km == 0 || s.tau == 0) {
    if (threadIdx.x == 0) {
      a.token[r] = km == 0 ? -1 : im;
      a.logprob[r] = km == 0 ? kNegInf : 0.f;
    }
    return;
  }
  q.wt.key_m = km;
  q.wt.m = (double)logit_of(km);
  q.wt.to_log2 = 1.4426950408889634074 / s.tau;
  q.wt.one = a.one;
  Cut cut{0, -1};
  u64 total = 0;
  bool known = false;  // total: the sum of the kept
  if (s.k < a.V) {
    cut = q.select(false, (double)s.k, &total);
    known = true;
  }
  if (s.p < 1) {
    if (!known) {
      u64 x = 0;
      q.each([&](int64_t, const uint32_t(&key)[kLoad]) {
#pragma unroll
        for (int u = 0; u < kLoad; ++u) x += q.wt.fix(q.wt.rel(key[u]));
      });
      total = block_sum64(x, s_sum);
    }
    const double limit = s.p * (double)total;
    u64 kept;
    const Cut c = q.select(true, limit > 0 ? limit : 0.5, &kept);
    // the shorter prefix
    if (c.key > cut.key || (c.key == cut.key && c.idx < cut.idx)) {
      cut = c;
      total = kept;
    }
    known = true;
  }
  auto weight = [&](uint32_t key, int64_t i) -> u64 {
    if (key == 0 || !cut.keeps(key, i)) return 0;
    const double w = q.wt.rel(key);
    return w >= s.min_p || key == km ? q.wt.fix(w) : 0;
  };
  if (!known || s.min_p > 0) {
    u64 x = 0;
    q.each([&](int64_t i0, const uint32_t(&key)[kLoad]) {
#pragma unroll
      for (int u = 0; u < kLoad; ++u) x += weight(key[u], i0 + u);
    });
    total = block_sum64(x, s_sum);
  }
  // (a whole sum exceeds u Z where it exceeds its whole part; total may need more bits than fp64 has)
  const double uz = s.u * (double)total;
  const u64 target = uz < (double)(total - 1) ? (u64)uz : total - 1;
  // the first token whose running sum exceeds the target
  u64 sum = 0;
#pragma unroll 1
  for (int64_t t0 = -q.lead; t0 < a.V; t0 += kTile) {
    const int64_t i0 = t0 + threadIdx.x * kLoad;
    uint32_t key[kLoad];
    load_keys(q.row, i0, a.V, key);
    u64 w[kLoad], x = 0;
#pragma unroll
    for (int u = 0; u < kLoad; ++u) x += w[u] = weight(key[u], i0 + u);
    u64 all;
    u64 at = sum + block_before64(x, s_sum, &all);
    sum += all;
    if (sum <= target) continue;
#pragma unroll
    for (int u = 0; u < kLoad; ++u) {
      const u64 before = at;
      at += w[u];
      if (before <= target && at > target) {
        a.token[r] = i0 + u;
        const double rel = key[u] == km ? 0.0 : ((double)logit_of(key[u]) - q.wt.m) / s.tau;
        a.logprob[r] = (float)(rel - log((double)total / a.one));
      }
    }
    break;
  }
}

}  // namespace

hipError_t sample_launch(int dtype, SampleParams p, hipStream_t stream) {
  if (p.R == 0) return hipSuccess;
  int bits = 0;
  while (bits < 31 && ((int64_t)1 << bits) < p.V) ++bits;
  p.one = (double)((int64_t)1 << (bits < 12 ? 50 : 62 - bits));
  timing_begin(kKindSample, stream);
  switch (dtype) {
    case kBF16: sample_row_kernel<bf16_t><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p); break;
    case kF16: sample_row_kernel<f16_t><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p); break;
    case kF32: sample_row_kernel<float><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p); break;
    default: return hipErrorInvalidValue;
  }
  timing_end(kKindSample, stream);
  return hipGetLastError();
}

}  // namespace swvr
