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

// Logits i0 .. i0 + L - 1 of a row (-inf outside 0 .. V - 1), in one load (fp32: 16 bytes each).  A row may begin
// anywhere: i0 + lead is a multiple of L, lead the row's distance from a border of L elements.
template <class T, int L>
__device__ __forceinline__ void load_logits(const T* row, int64_t i0, int64_t V, float (&x_)[L]) {
  if (i0 >= 0 && i0 + L <= V) {
    struct alignas(L * sizeof(T) < 16 ? L * sizeof(T) : 16) X {
      T v[L];
    };
    const X x = *reinterpret_cast<const X*>(row + i0);
#pragma unroll
    for (int u = 0; u < L; ++u) x_[u] = (float)x.v[u];
  } else {
#pragma unroll
    for (int u = 0; u < L; ++u) x_[u] = i0 + u >= 0 && i0 + u < V ? (float)row[i0 + u] : kNegInf;
  }
}
template <class T, int L>
__device__ __forceinline__ void load_keys(const T* row, int64_t i0, int64_t V, uint32_t (&key)[L]) {
  float x[L];
  load_logits(row, i0, V, x);
#pragma unroll
  for (int u = 0; u < L; ++u) key[u] = key_of(x[u]);
}

// Weights of a row: w = 2^t, t = (l - m) to_log2, to_log2 = log2(e) / tau, in fp64: with n the whole number next to
// 32 t and f = t - n / 32, 2^t = 2^(n / 32) e^(f ln 2), the first from a table of 2^(i / 32) in LDS and an exponent,
// the second's Taylor series to the 4th power (|f| <= 1/64: off by 1.2e-12 of itself; t is rounded by 7e-15 at -45).
// A random error e of every w moves the running sums by about e / sqrt(n) of themselves for n tokens, and there are
// n borders: a token differs from exact arithmetic's in one of 1 / (e sqrt(n)) draws, 2e9 for n = 151936.
constexpr int kPowers = 32;
__device__ __forceinline__ void fill_powers(double* s) {  // no barrier
  if (threadIdx.x < kPowers) s[threadIdx.x] = exp2((double)threadIdx.x / kPowers);
}
struct Weigh {
  const double* powers;  // [kPowers], LDS
  double m, to_log2, one;  // one: 2^shift
  float m_f;
  uint32_t key_m;
  __device__ __forceinline__ double rel(uint32_t key) const { return rel(logit_of(key)); }
  __device__ __forceinline__ double rel(float l) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: sums with it are whole numbers, in the low bits
    const double t = ((double)l - m) * to_log2;
    const double y = fma(t, (double)kPowers, kRound);
    const int n = (int)__double_as_longlong(y);
    const double f = fma(y - kRound, -1.0 / kPowers, t);
    double x = 0.009618129107628477;  // ln(2)^4 / 4!, ...
    x = fma(x, f, 0.05550410866482158);
    x = fma(x, f, 0.24022650695910072);
    x = fma(x, f, 0.6931471805599453);
    x = fma(x, f, 1.0);
    const double w = x * __longlong_as_double(__double_as_longlong(powers[n & (kPowers - 1)]) +
                                              ((long long)(n >> 5) << 52));
    // (t is NaN for a NaN, and where the largest logit is infinite for tokens equal to it)
    return l == m_f ? 1.0 : t > -1000 ? w : 0.0;
  }
  // w in units of 2^-shift, to nearest: below 2^52, so the sum's low bits are the whole number
  __device__ __forceinline__ u64 fix(double w) const {
    return (u64)__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

// x of the lane that DPP control CTRL names, 0 where there is none or the row is not in RM.
template <int CTRL, int RM = 0xf>
__device__ __forceinline__ u64 dpp64(u64 x) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, RM, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, RM, 0xf, false);
  return (u64)(uint32_t)hi << 32 | (uint32_t)lo;
}
// Inclusive scan over the wave under an operation with identity 0: within rows of 16 lanes (row_shr 1, 2, 4, 8),
// then the last lane of row 0 and 2 into rows 1 and 3 (row_bcast 15), and lane 31 into the upper half (row_bcast 31).
// (DPP moves cost a few cycles where __shfl goes through LDS: a workgroup's scan of 1024 threads 0.85 -> 0.5 us.)
template <class Op>
__device__ __forceinline__ u64 wave_scan64(u64 x, Op op) {
  x = op(x, dpp64<0x111>(x));
  x = op(x, dpp64<0x112>(x));
  x = op(x, dpp64<0x114>(x));
  x = op(x, dpp64<0x118>(x));
  x = op(x, dpp64<0x142, 0xa>(x));
  return op(x, dpp64<0x143, 0xc>(x));
}
struct Sum64 {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max64 {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};
__device__ __forceinline__ u64 last_lane64(u64 x) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
}
__device__ __forceinline__ u64 wave_sum64(u64 x) { return last_lane64(wave_scan64(x, Sum64())); }
__device__ __forceinline__ u64 wave_max64(u64 x) { return last_lane64(wave_scan64(x, Max64())); }

// Sum over a workgroup of NW waves, in every thread; s: NW words of LDS, free again at the next barrier after.
template <int NW>
__device__ __forceinline__ u64 block_sum64(u64 x, u64* s) {
  x = wave_sum64(x);
  __syncthreads();
  if (lane_id() == 0) s[wave_id()] = x;
  __syncthreads();
  x = 0;
#pragma unroll 4
  for (int j = 0; j < NW; ++j) x += s[j];
  return x;
}

// Sum of the threads before this one, and of all (total).
template <int NW>
__device__ __forceinline__ u64 block_before64(u64 x, u64* s, u64* total) {
  const u64 y = wave_scan64(x, Sum64());
  __syncthreads();
  if (lane_id() == 63) s[wave_id()] = y;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll 4
  for (int j = 0; j < NW; ++j) {
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
  s.min_p = s.min_p > 0 ? (s.min_p < 1 ? s.min_p : 1) : 0;  // (at 1 the largest, whose w is 1, are left)
  return s;
}

// ---------------------------------------------------------------- a row by one workgroup
// Passes over the row: the maximum; for top-k and top-p each, the cut by radix descent over the 32 key bits (11, 11
// and 10 bits: a histogram of counts and weights, the bin where the count reaches k or the weight p Z_k), then the
// place of the last kept one among equal logits; the kept sum; and the running sum up to the token.  For rows too
// long for the launches below, for k above kTopK and for lists that overflow: up to 9 reads of the row by one CU, whose
// arithmetic and barriers bound it (a row of 151936 in bf16 with top-k 5000 and top-p: 420 us; top-k 50 takes 18).
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
      const u64 bw = above_w + block_before64<kRowWaves>(w1 + w0, s_sum, &all_w);
      const u64 bn = above_n + block_before64<kRowWaves>(n1 + n0, s_sum, &all_n);
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
      u64 at = seen + block_before64<kRowWaves>(n, s_sum, &all);
#pragma unroll
      for (int u = 0; u < kLoad; ++u)
        if (key[u] == lo && ++at == take) s_out[0] = (u64)(i0 + u);
      seen += all;
    }
    __syncthreads();
    return Cut{lo, (int64_t)s_out[0]};
  }
};

// Words of LDS of a row's workgroup.
struct RowShared {
  u64* sum;       // [kRowWaves]
  u64* out;       // [4]
  u64* w;         // [kBins]
  uint32_t* cnt;  // [kBins]
};

// The token of row r, whose largest logit is in wt (not -inf) and whose temperature is not 0.
template <class T>
__device__ void sample_row(const SampleParams& a, int64_t r, const RowSettings& s, const Weigh& wt, RowShared sh) {
  RowSampler<T> q;
  q.row = static_cast<const T*>(a.logits) + r * a.ld;
  q.V = a.V;
  q.lead = (int)((reinterpret_cast<uintptr_t>(q.row) / sizeof(T)) % kLoad);
  q.wt = wt;
  q.s_sum = sh.sum;
  q.s_w = sh.w;
  q.s_cnt = sh.cnt;
  q.s_out = sh.out;
  u64* const s_sum = sh.sum;
  const uint32_t km = wt.key_m;
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
      total = block_sum64<kRowWaves>(x, s_sum);
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
    return w >= s.min_p ? q.wt.fix(w) : 0;
  };
  if (!known || s.min_p > 0) {
    u64 x = 0;
    q.each([&](int64_t i0, const uint32_t(&key)[kLoad]) {
#pragma unroll
      for (int u = 0; u < kLoad; ++u) x += weight(key[u], i0 + u);
    });
    total = block_sum64<kRowWaves>(x, s_sum);
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
    u64 at = sum + block_before64<kRowWaves>(x, s_sum, &all);
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

// A token whose place in the order is its key and then its index, as one number: larger is earlier; 0: nothing.
__device__ __forceinline__ u64 place_of(uint32_t key, int64_t i) {
  return key == 0 ? 0 : (u64)key << 32 | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ uint32_t key_at(u64 place) { return (uint32_t)(place >> 32); }
__device__ __forceinline__ int64_t index_at(u64 place) { return (int64_t)(uint32_t)~(uint32_t)place; }
__device__ __forceinline__ Weigh weigh_of(const SampleParams& a, const RowSettings& s, uint32_t key_m,
                                          const double* powers) {
  Weigh w;
  w.powers = powers;
  w.m_f = logit_of(key_m);
  w.m = (double)w.m_f;
  w.to_log2 = 1.4426950408889634074 / s.tau;
  w.one = a.one;
  w.key_m = key_m;
  return w;
}

// Writes the token of a row that needs no draw: none, or at temperature 0 the first in order.
__device__ __forceinline__ bool settled(const SampleParams& a, int64_t r, const RowSettings& s, u64 first) {
  if (first != 0 && s.tau != 0) return false;
  if (threadIdx.x == 0) {
    a.token[r] = first == 0 ? -1 : index_at(first);
    a.logprob[r] = first == 0 ? kNegInf : 0.f;
  }
  return true;
}

// ---- a row in one launch
template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(SampleParams a) {
  __shared__ u64 s_sum[kRowWaves], s_w[kBins], s_out[4];
  __shared__ double s_powers[kPowers];
  __shared__ uint32_t s_cnt[kBins];
  fill_powers(s_powers);
  const int64_t r = blockIdx.x;
  const RowSettings s = settings_of(a, r);
  const T* const row = static_cast<const T*>(a.logits) + r * a.ld;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kLoad);
  u64 first = 0;
#pragma unroll 1
  for (int64_t i0 = (int64_t)threadIdx.x * kLoad - lead; i0 < a.V; i0 += kTile) {
    uint32_t key[kLoad];
    load_keys(row, i0, a.V, key);
#pragma unroll
    for (int u = 0; u < kLoad; ++u) {
      const u64 x = place_of(key[u], i0 + u);
      first = x > first ? x : first;
    }
  }
  first = wave_max64(first);
  if (lane_id() == 0) s_sum[wave_id()] = first;
  __syncthreads();
#pragma unroll 4
  for (int j = 0; j < kRowWaves; ++j) first = s_sum[j] > first ? s_sum[j] : first;
  if (settled(a, r, s, first)) return;
  sample_row<T>(a, r, s, weigh_of(a, s, key_at(first), s_powers), RowShared{s_sum, s_out, s_w, s_cnt});
}

// ---------------------------------------------------------------- a row by many workgroups
// Rows of more than kRowMost logits, in up to four launches for all of them:
//   sample_max_kernel    per sub-block of kSub logits (a wave each) its first token in order, and per group of
//                        2^gshift logits (up to kGroups groups a row) its largest key;
//   sample_hist_kernel   rows with top-p alone: the weight per bin of the distance from the largest logit;
//   sample_sums_kernel   rows without top-k: per sub-block, the weight of the tokens before the bin in which the
//                        prefix of p Z ends; that bin's own tokens go to the row's list;
//   sample_finish_kernel the token.  With top-k, the k-th largest of the groups' largest keys is a bound that at least
//                        k tokens reach, and, the largest tokens lying scattered, few more: only the groups that
//                        reach it are read again, and their tokens that do are the row's list.  The cut is found
//                        in the list from counts and weights per bin (draw_row), then the sub-block that holds the
//                        drawn token, which is read again.
// So a row is read once with top-k, twice with min-p or nothing, three times with top-p, and its logits never sorted.
// A list that would pass kList tokens, or kSegList from one workgroup (equal logits, a nearly flat row), leaves its
// row to sample_row, in the same launch, as does a k above kTopK.  Every sum is one of whole numbers, so its order
// does not matter.
constexpr int kSub = 2048, kGroups = 4096, kList = 4096, kSegList = 2048, kTopK = 1024, kFew = 128,
              kDense = 512, kHistWaves = 8;
constexpr int64_t kRowMost = 4096, kStagedMost = ((int64_t)1 << 21) - 8;  // (groups of at most a wave's 512)
constexpr int kSubsMost = (int)(((int64_t)1 << 21) / kSub);
constexpr int kWaveLoad = 8, kCross = 3;

enum RowKind { kGreedy, kTopKRow, kTopPRow, kSumRow, kWholeRow };
__device__ __forceinline__ RowKind kind_of(const RowSettings& s, int64_t V) {
  return s.tau == 0 ? kGreedy : s.k < V ? (s.k <= kTopK ? kTopKRow : kWholeRow) : s.p < 1 ? kTopPRow : kSumRow;
}

struct Staged {
  SampleParams a;
  int64_t r0;       // first row of this launch
  int n_sub;        // sub-blocks of a row
  int gshift;       // log2 of a group's logits
  int n_seg;        // workgroups of 4 waves per row (of the histogram, kHistWaves)
  u64* first;       // [rows][n_sub] place_of the sub-block's first token in order
  uint32_t* group;  // [rows][kGroups] largest keys
  u64* hist;        // [rows][kBins] weights
  u64* list;        // [rows][kList] places
  int* n_list;      // [rows]
  u64* sums;        // [rows][n_sub]
  u64* crossing;    // [rows][kCross]: the bin in which the prefix ends, the weight before it, the whole weight
  int may_k, may_p, may_sum;  // whether a row may have top-k, top-p alone, no top-k (the host cannot see every setting)
};

template <class T>
struct RowView {
  const T* row;
  int64_t V;
  int lead;
  __device__ __forceinline__ RowView(const SampleParams& a, int64_t r)
      : row(static_cast<const T*>(a.logits) + r * a.ld), V(a.V) {
    lead = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kWaveLoad);
  }
};

// Room for this lane's c entries at the end of a list of *n (LDS), in one atomic of the whole wave.
__device__ __forceinline__ int append(int* n, int c) {
  const int to = (int)wave_scan64((u64)c, Sum64());
  int base = 0;
  if (lane_id() == 63 && to > 0) base = atomicAdd(n, to);
  return __builtin_amdgcn_readlane(base, 63) + to - c;
}

// kWaveLoad consecutive logits of a lane from i0 on (i0 + lead a multiple of kWaveLoad), as stored: loads of several go
// out before the first is used (converted inside the branch of load_logits, each waited for the one before: the first
// launch took 42 us for 512 rows of 151936).  Where they reach over an end of the row, fix() replaces them.
template <class T>
struct alignas(kWaveLoad * sizeof(T) < 16 ? kWaveLoad * sizeof(T) : 16) Chunk {
  T v[kWaveLoad];
};
template <class T>
__device__ __forceinline__ Chunk<T> load_chunk(const RowView<T>& v, int64_t i0) {
  // the nearest chunk inside the row (V > 2 kWaveLoad)
  const int64_t lo = v.lead == 0 ? 0 : kWaveLoad - v.lead;
  const int64_t hi = lo + (v.V - lo) / kWaveLoad * kWaveLoad - kWaveLoad;
  const int64_t at = i0 < lo ? lo : i0 > hi ? hi : i0;
  return *reinterpret_cast<const Chunk<T>*>(v.row + at);
}
template <class T>
__device__ __forceinline__ void chunk_logits(const RowView<T>& v, int64_t i0, const Chunk<T>& c, float (&x)[kWaveLoad]) {
#pragma unroll
  for (int u = 0; u < kWaveLoad; ++u) x[u] = (float)c.v[u];
  if (i0 < 0 || i0 + kWaveLoad > v.V)
#pragma unroll
    for (int u = 0; u < kWaveLoad; ++u) x[u] = i0 + u >= 0 && i0 + u < v.V ? (float)v.row[i0 + u] : kNegInf;
}

// The logits of a wave's sub-block, step j of kSteps holding kWaveLoad consecutive ones of each lane from first(j) on
// (outside the row: -inf).
constexpr int kSteps = kSub / (64 * kWaveLoad);
template <class T>
struct SubBlock {
  int sub;
  int64_t i0;
  Chunk<T> c[kSteps];
  __device__ __forceinline__ SubBlock(const Staged& p, const RowView<T>& v, int seg, int waves) {
    sub = seg * waves + wave_id();
    i0 = (int64_t)sub * kSub - v.lead + lane_id() * kWaveLoad;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) c[j] = load_chunk(v, first(j));
  }
  __device__ __forceinline__ int64_t first(int j) const { return i0 + j * 64 * kWaveLoad; }
};

// A row's first token in order, by each wave for itself.
__device__ __forceinline__ u64 row_first(const Staged& p, int64_t q) {
  u64 first = 0;
  for (int i = lane_id(); i < p.n_sub; i += 64) {
    const u64 x = p.first[q * p.n_sub + i];
    first = x > first ? x : first;
  }
  return wave_max64(first);
}

// Bin of a key: its distance below the largest in units of 46 log2-steps of weight / kBins, in fp32: no smaller for a
// smaller logit.  The last bin takes everything farther away too: weights of 0, but in rows of up to 65536 logits, whose
// weights have 46 to 49 bits.
__device__ __forceinline__ float bin_scale(const Weigh& w) { return (float)(w.to_log2 * (kBins / 46.0)); }
__device__ __forceinline__ int bin_of(float l, const Weigh& w, float scale) {
  const float x = (w.m_f - l) * scale;
  return l == w.m_f ? 0 : x < kBins - 1 ? (int)x : kBins - 1;
}

// Bound by memory: 512 rows of 151936 in bf16 (156 MB) in 34 us, 4.6 TB/s.
template <class T>
__global__ __launch_bounds__(256) void sample_max_kernel(Staged p) {
  const int64_t q = blockIdx.x / p.n_seg, r = p.r0 + q;
  const RowSettings s = settings_of(p.a, r);
  const RowKind kind = kind_of(s, p.a.V);
  const int seg = (int)(blockIdx.x % p.n_seg);
  if (kind == kTopPRow) {
    for (int i = seg * 256 + threadIdx.x; i < kBins; i += 256 * p.n_seg) p.hist[q * kBins + i] = 0;
    if (seg == 0 && threadIdx.x == 0) p.n_list[q] = 0;
  }
  const int lanes = 1 << (p.gshift - 3);  // of a group
  const RowView<T> v(p.a, r);
  const SubBlock<T> b(p, v, (int)(blockIdx.x % p.n_seg), 4);
  if (b.sub >= p.n_sub) return;
  u64 first = 0;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    uint32_t k = 0;
    int at = 0;
    float l[kWaveLoad];
    chunk_logits(v, b.first(j), b.c[j], l);
#pragma unroll
    for (int u = 0; u < kWaveLoad; ++u) {
      const uint32_t key = key_of(l[u]);
      at = key > k ? u : at;
      k = key > k ? key : k;
    }
    const u64 x = place_of(k, b.first(j) + at);
    first = x > first ? x : first;
    if (kind != kTopKRow) continue;
    for (int o = 1; o < lanes; o <<= 1) {
      const uint32_t y = __shfl_xor(k, o);
      k = y > k ? y : k;
    }
    if ((lane_id() & (lanes - 1)) == 0)
      p.group[q * kGroups + (((int64_t)b.sub * kSub + (j * 64 + lane_id()) * kWaveLoad) >> p.gshift)] = k;
  }
  first = wave_max64(first);
  if (lane_id() == 0) p.first[q * p.n_sub + b.sub] = first;
}

// Bound by its arithmetic, some 30 fp64 and integer instructions and an LDS add for each logit: 102 us for 512 rows of
// 151936.  (Of 4 waves, which add twice as many bins to the rows', 110; 16 leave fewer at work at its barriers: on a
// third as many rows 47 us for the 40 of 4.)
template <class T>
__global__ __launch_bounds__(64 * kHistWaves) void sample_hist_kernel(Staged p) {
  __shared__ u64 s_hist[kBins];
  __shared__ double s_powers[kPowers];
  const int n_seg = (p.n_sub + kHistWaves - 1) / kHistWaves;
  const int64_t q = blockIdx.x / n_seg, r = p.r0 + q;
  const RowSettings s = settings_of(p.a, r);
  if (kind_of(s, p.a.V) != kTopPRow) return;
  const RowView<T> v(p.a, r);
  const SubBlock<T> b(p, v, (int)(blockIdx.x % n_seg), kHistWaves);
  const u64 first = row_first(p, q);
  if (first == 0) return;
  fill_powers(s_powers);
  for (int i = threadIdx.x; i < kBins; i += 64 * kHistWaves) s_hist[i] = 0;
  __syncthreads();
  const Weigh wt = weigh_of(p.a, s, key_at(first), s_powers);
  const float scale = bin_scale(wt);
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float l[kWaveLoad];
    chunk_logits(v, b.first(j), b.c[j], l);
#pragma unroll
    for (int u = 0; u < kWaveLoad; ++u) {
      const u64 w = wt.fix(wt.rel(l[u]));
      if (w) atomicAdd(&s_hist[bin_of(l[u], wt, scale)], w);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += 64 * kHistWaves)
    if (s_hist[i]) atomicAdd(&p.hist[q * kBins + i], s_hist[i]);
}

// As the histogram, with its bins read by every workgroup (16 KB, from L2), but few logits are in the prefix: they are
// gathered in LDS and only they are weighed (121 us for those rows with all of them weighed, so 83).
template <class T>
__global__ __launch_bounds__(256) void sample_sums_kernel(Staged p) {
  __shared__ u64 s_sum[4], s_cross[kCross], s_list[kSegList];
  __shared__ float s_dense[4][kDense];
  __shared__ double s_powers[kPowers];
  __shared__ int s_n, s_at;
  const int64_t q = blockIdx.x / p.n_seg, r = p.r0 + q;
  const RowSettings s = settings_of(p.a, r);
  const RowKind kind = kind_of(s, p.a.V);
  if (kind != kTopPRow && kind != kSumRow) return;
  const RowView<T> v(p.a, r);
  const SubBlock<T> b(p, v, (int)(blockIdx.x % p.n_seg), 4);
  const u64 first = row_first(p, q);
  if (first == 0) return;
  fill_powers(s_powers);
  if (threadIdx.x == 0) s_n = 0;
  int cross = kBins;
  if (kind == kTopPRow) {
    constexpr int kPer = kBins / 256;
    u64 w[kPer], sum = 0, total;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += w[i] = p.hist[q * kBins + threadIdx.x * kPer + i];
    u64 at = block_before64<4>(sum, s_sum, &total);
    const double pz = s.p * (double)total, limit = pz > 0 ? pz : 0.5;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (w[i] && (double)at < limit && (double)(at + w[i]) >= limit) {
        s_cross[0] = threadIdx.x * kPer + i;
        s_cross[1] = at;
        s_cross[2] = total;
      }
      at += w[i];
    }
    __syncthreads();
    cross = (int)s_cross[0];
    if (blockIdx.x % p.n_seg == 0 && threadIdx.x < kCross)
      p.crossing[q * kCross + threadIdx.x] = s_cross[threadIdx.x];
  }
  __syncthreads();
  const Weigh wt = weigh_of(p.a, s, key_at(first), s_powers);
  const float scale = bin_scale(wt);
  u64 sum = 0;
  uint32_t hits = 0, in = 0;  // a bit for each of this lane's tokens in the bin; in the prefix before it
  int n_in = kDense + 1;
  if (kind == kTopPRow) {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      float x[kWaveLoad];
      chunk_logits(v, b.first(j), b.c[j], x);
#pragma unroll
      for (int u = 0; u < kWaveLoad; ++u) {
        const int bin = bin_of(x[u], wt, scale);
        in |= bin < cross ? 1u << (j * kWaveLoad + u) : 0u;
        hits |= (bin == cross && x[u] > kNegInf) ? 1u << (j * kWaveLoad + u) : 0u;
        asm volatile("" : "+v"(hits), "+v"(in));  // (for registers, as below: 105 us, so 83)
      }
    }
    const int to = (int)wave_scan64((u64)__popc(in), Sum64());
    n_in = __builtin_amdgcn_readlane(to, 63);
    if (n_in <= kDense) {
      // few of the sub-block: gathered, so that only they are weighed
      float* const dense = s_dense[wave_id()];
      int at = to - __popc(in);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        float x[kWaveLoad];
        chunk_logits(v, b.first(j), b.c[j], x);
#pragma unroll
        for (int u = 0; u < kWaveLoad; ++u)
          if (in >> (j * kWaveLoad + u) & 1) {
            dense[at] = x[u];
            ++at;
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int i = lane_id(); i < n_in; i += 64) {
        const double w = wt.rel(dense[i]);
        sum += w >= s.min_p ? wt.fix(w) : 0;
      }
    }
  }
  if (n_in > kDense) {
    // (one element after another: left to it, the compiler keeps all 32 in flight, in 245 registers, 75 us for 50)
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      float x[kWaveLoad];
      chunk_logits(v, b.first(j), b.c[j], x);
#pragma unroll
      for (int u = 0; u < kWaveLoad; ++u) {
        const double w = wt.rel(x[u]);
        const bool mine = kind != kTopPRow || (in >> (j * kWaveLoad + u) & 1);
        sum += mine && w >= s.min_p ? wt.fix(w) : 0;
        asm volatile("" : "+v"(sum));
      }
    }
  }
  // the bin's tokens, few, are read again (kept apart, they hold no registers)
  for (; hits != 0; hits &= hits - 1) {
    const int i = __ffs((int)hits) - 1;
    const int64_t at = b.first(i / kWaveLoad) + i % kWaveLoad;
    const int n = atomicAdd(&s_n, 1);
    if (n < kSegList) s_list[n] = place_of(key_of((float)v.row[at]), at);
  }
  sum = wave_sum64(sum);
  if (lane_id() == 0 && b.sub < p.n_sub) p.sums[q * p.n_sub + b.sub] = sum;
  if (kind != kTopPRow) return;
  // the bin's tokens of this workgroup to the row's list, whose order does not matter
  __syncthreads();
  const int n = s_n;
  if (threadIdx.x == 0 && n > 0) s_at = atomicAdd(&p.n_list[q], n <= kSegList ? n : kList + 1);
  __syncthreads();
  for (int i = threadIdx.x; i < n && n <= kSegList; i += 256)
    if (s_at + i < kList) p.list[q * kList + s_at + i] = s_list[i];
}

// Bin of a key's distance d below the largest: 64 per octave of d (the upper bits of d as a float), so that the
// largest keys, whatever they are, spread over many.
constexpr uint32_t kOneBits = 127u << 6;  // 1.f's upper bits
__device__ __forceinline__ int distance_bin(uint32_t d) {
  const uint32_t x = d == 0 ? 0 : (__float_as_uint((float)d) >> 17) - kOneBits;
  return x < kBins ? (int)x : kBins - 1;
}

// LDS of a row's last workgroup.
struct FinishShared {
  u64 *list, *w, *sub, *sum, *out;  // [kList], [kList], [kSubsMost], [kRowWaves], [6]
  int *n, *m;
};

// The token of row r from its list of n tokens (in LDS, after a barrier): with kTopKRow all that it keeps are in there,
// with kTopPRow those of the bin in which its prefix ends, with kSumRow none; sub: the sums of sub-blocks
// 2 threadIdx.x and the next (not with kTopKRow), crossing: as in Staged.
template <class T>
__device__ __forceinline__ void draw_row(const SampleParams& a, int64_t r, const RowSettings& s, const RowView<T>& v,
                                         const Weigh& wt, RowKind kind, int n, int n_sub, u64 (&sub)[2],
                                         const u64 (&crossing)[kCross], const FinishShared& sh) {
  u64 *const s_list = sh.list, *const s_w = sh.w, *const s_sub = sh.sub, *const s_sum = sh.sum, *const s_out = sh.out;
  int *const s_n = sh.n, *const s_m = sh.m;
  constexpr int kPer = kList / kRowThreads;  // list entries of a thread
  const int j0 = 2 * threadIdx.x;
  auto draw = [&](u64 place, u64 total) {  // by one thread
    const uint32_t key = key_at(place);
    const double rel = key == wt.key_m ? 0.0 : ((double)logit_of(key) - wt.m) / s.tau;
    a.token[r] = index_at(place);
    a.logprob[r] = (float)(rel - log((double)total / a.one));
  };
  auto target_of = [&](u64 total) {
    const double uz = s.u * (double)total;
    return uz < (double)(total - 1) ? (u64)uz : total - 1;
  };
  if (kind == kTopKRow && n <= kFew) {
    // few tokens, by one wave without barriers: each against all, for its place in the order and the weight before
    // it, then for the kept weight before it by index
    if (wave_id() != 0) return;
    const int lane = lane_id();
    u64 place[2], w[2], at[2] = {0, 0};
    double rel[2];
    int rank[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      place[i] = lane + 64 * i < n ? s_list[lane + 64 * i] : 0;
      rel[i] = place[i] != 0 ? wt.rel(key_at(place[i])) : 0;
      s_w[lane + 64 * i] = w[i] = wt.fix(rel[i]);
    }
    if (lane < 4) s_list[n + lane] = s_w[kFew + lane] = 0;  // to a multiple of 4
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int j = 0; j < n; j += 4)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const u64 y = s_list[j + u], wy = s_w[j + u];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          rank[i] += y > place[i];
          at[i] += y > place[i] ? wy : 0;
        }
      }
    u64 z = 0, total = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) z += place[i] != 0 && rank[i] < s.k ? w[i] : 0;
    z = wave_sum64(z);
    const double pz = s.p < 1 ? s.p * (double)z : kPosInf, limit = pz > 0 ? pz : 0.5;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool keep = place[i] != 0 && rank[i] < s.k && (double)at[i] < limit && rel[i] >= s.min_p;
      w[i] = keep ? w[i] : 0;
      s_w[lane + 64 * i] = w[i];
      total += w[i];
      at[i] = 0;
    }
    total = wave_sum64(total);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int j = 0; j < n; j += 4)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const u64 y = s_list[j + u], wy = s_w[j + u];
#pragma unroll
        for (int i = 0; i < 2; ++i) at[i] += (uint32_t)y > (uint32_t)place[i] ? wy : 0;
      }
    const u64 target = target_of(total);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (at[i] <= target && at[i] + w[i] > target) draw(place[i], total);
    return;
  }
  u64 cut = 0;  // the last token of the prefix (0: every token)
  for (int i = threadIdx.x; i < n_sub; i += kRowThreads) s_sub[i] = 0;
  if (n > 0) {
    // The cut: counts and weights of the list's tokens per bin of their distance below the largest key; with top-k the
    // bin in which the k-th lies (where the list has more), and in it the cut and the weight up to it; then the bin in
    // which the weight passes the limit of top-p.  A bin holds few tokens, each compared with all, or is split again.
    const u64 before_list = kind == kTopPRow ? crossing[1] : 0;
    u64* const bin_w = s_w;                                                     // [kBins]
    uint32_t* const bin_n = reinterpret_cast<uint32_t*>(s_w + kBins);           // [kBins]
    u64* const few = s_w + kBins + kBins / 2;                                   // [kFew] places, then weights
    if (threadIdx.x == 0) *s_n = *s_m = 0;
    for (int i = threadIdx.x; i < kBins + kBins / 2; i += kRowThreads) s_w[i] = 0;
    __syncthreads();
    // (its tokens stay in LDS: the registers are needed below)
    auto place = [&](int i) -> u64 {
      const int at = threadIdx.x + i * kRowThreads;
      return at < n ? s_list[at] : 0;
    };
    auto bin_of_place = [&](u64 x) { return distance_bin(wt.key_m - key_at(x)); };
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const u64 x = place(i);
      if (x == 0) continue;
      const u64 w = wt.fix(wt.rel(key_at(x)));
      atomicAdd(&bin_n[bin_of_place(x)], 1u);
      if (w) atomicAdd(&bin_w[bin_of_place(x)], w);
    }
    __syncthreads();
    const u64 w0 = bin_w[j0], w1 = bin_w[j0 + 1];
    const uint32_t n0 = bin_n[j0], n1 = bin_n[j0 + 1];
    u64 all_w, all_n;
    const u64 at_w = before_list + block_before64<kRowWaves>(w0 + w1, s_sum, &all_w);
    const uint32_t at_n = (uint32_t)block_before64<kRowWaves>(n0 + n1, s_sum, &all_n);
    const uint32_t k = kind == kTopKRow && s.k < (int64_t)all_n ? (uint32_t)s.k : (uint32_t)all_n;
    double limit = kPosInf;
    // In a bin: the prefix ends in the last one that begins inside both limits.
    auto ends = [&](uint32_t n_at, u64 w_at, uint32_t in_n, u64 in_w) {
      return in_n > 0 && n_at < k && (double)w_at < limit && (n_at + in_n >= k || (double)(w_at + in_w) >= limit);
    };
    auto mark = [&](int bin, uint32_t n_at, u64 w_at, uint32_t in_n) {
      s_out[0] = bin;
      s_out[1] = w_at;
      s_out[2] = n_at;
      s_out[3] = in_n;
    };
    // the count's cut, then the weight's
    u64 kept = all_w;
#pragma unroll 1
    for (int by_weight = k < all_n ? 0 : 1; by_weight < (kind == kTopPRow || s.p < 1 ? 2 : 1); ++by_weight) {
      if (by_weight) {
        const double pz = s.p * (double)(kind == kTopPRow ? crossing[2] : kept);
        limit = pz > 0 ? pz : 0.5;
      }
      if (ends(at_n, at_w, n0, w0)) mark(j0, at_n, at_w, n0);
      else if (ends(at_n + n0, at_w + w0, n1, w1)) mark(j0 + 1, at_n + n0, at_w + w0, n1);
      if (threadIdx.x == 0) s_out[4] = s_out[5] = 0;
      __syncthreads();
      int m = (int)s_out[3];
      u64 b_w = s_out[1];
      uint32_t b_n = (uint32_t)s_out[2];
      uint32_t here = 0;  // a bit for each of this thread's tokens that is in the bin
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const u64 x = place(i);
        here |= x != 0 && bin_of_place(x) == (int)s_out[0] ? 1u << i : 0u;
      }
      // Too many to compare (near or equal logits): bins over the range of their places, which narrows by 2^10 or
      // more each time, so at most 6 times.  (Sorting the list instead: 48 rows of 128256 with top-p 60 us, so 53.)
      while (m > kFew) {
        u64 top = 0, low = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const u64 x = place(i);
          top = (here >> i & 1) && x > top ? x : top;
          low = (here >> i & 1) && ~x > low ? ~x : low;
        }
        top = wave_max64(top);
        low = wave_max64(low);
        if (lane_id() == 0) {
          atomicMax(&s_out[4], top);
          atomicMax(&s_out[5], low);
        }
        for (int i = threadIdx.x; i < kBins + kBins / 2; i += kRowThreads) s_w[i] = 0;
        __syncthreads();
        top = s_out[4];
        low = ~s_out[5];
        const float scale = (float)(kBins - 1) / (float)(top - low);
        auto bin_here = [&](u64 x) { return min(kBins - 1, (int)((float)(top - x) * scale)); };
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (here >> i & 1) {
            const u64 x = place(i);
            atomicAdd(&bin_n[bin_here(x)], 1u);
            atomicAdd(&bin_w[bin_here(x)], wt.fix(wt.rel(key_at(x))));
          }
        __syncthreads();
        const u64 x0 = bin_w[j0], x1 = bin_w[j0 + 1];
        const uint32_t c0 = bin_n[j0], c1 = bin_n[j0 + 1];
        u64 all;
        const u64 x_at = b_w + block_before64<kRowWaves>(x0 + x1, s_sum, &all);
        const uint32_t c_at = b_n + (uint32_t)block_before64<kRowWaves>(c0 + c1, s_sum, &all);
        if (ends(c_at, x_at, c0, x0)) mark(j0, c_at, x_at, c0);
        else if (ends(c_at + c0, x_at + x0, c1, x1)) mark(j0 + 1, c_at + c0, x_at + x0, c1);
        if (threadIdx.x == 0) s_out[4] = s_out[5] = 0;
        __syncthreads();
        m = (int)s_out[3];
        b_w = s_out[1];
        b_n = (uint32_t)s_out[2];
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if ((here >> i & 1) && bin_here(place(i)) != (int)s_out[0]) here &= ~(1u << i);
      }
      // each against all, by the first wave
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (here >> i & 1) few[atomicAdd(s_m, 1)] = place(i);
      __syncthreads();
      if (wave_id() == 0) {
        const int lane = lane_id();
        u64 x[2], y[2], at[2] = {b_w, b_w};
        uint32_t rank[2] = {b_n, b_n};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[i] = lane + 64 * i < m ? few[lane + 64 * i] : 0;
          y[i] = x[i] != 0 ? wt.fix(wt.rel(key_at(x[i]))) : 0;
          few[kFew + lane + 64 * i] = y[i];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
        for (int j = 0; j < m; ++j) {
          const u64 z = few[j], wz = few[kFew + j];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            rank[i] += z > x[i];
            at[i] += z > x[i] ? wz : 0;
          }
        }
        u64 last = ~0ull, sum = 0;  // the smallest place of the prefix
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool kept = x[i] != 0 && rank[i] < k && (double)at[i] < limit;
          last = kept && x[i] < last ? x[i] : last;
          sum += kept ? y[i] : 0;
        }
        last = ~wave_max64(~last);
        sum = wave_sum64(sum);
        if (lane == 0) {
          s_out[0] = last;
          s_out[1] = b_w + sum;
          *s_m = 0;
        }
      }
      __syncthreads();
      cut = s_out[0];
      kept = s_out[1];
      __syncthreads();
    }
    // the prefix's tokens join the sub-blocks' sums (with top-k they are all there is)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const u64 x = place(i);
      if (x == 0 || x < cut) continue;
      const double rel = wt.rel(key_at(x));
      const u64 w = rel >= s.min_p ? wt.fix(rel) : 0;
      if (w) atomicAdd(&s_sub[(index_at(x) + v.lead) / kSub], w);
    }
  }
  // the sub-block that holds the token, then its place there
  __syncthreads();
  u64 total;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (kind == kTopKRow) sub[i] = 0;
    if (j0 + i < n_sub) sub[i] += s_sub[j0 + i];
  }
  u64 at = block_before64<kRowWaves>(sub[0] + sub[1], s_sum, &total);
  const u64 target = target_of(total);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (at <= target && at + sub[i] > target) {
      s_out[0] = j0 + i;
      s_out[1] = at;
    }
    at += sub[i];
  }
  __syncthreads();
  const int64_t i0 = (int64_t)s_out[0] * kSub - v.lead + 2 * threadIdx.x;
  at = s_out[1];
  u64 place[2], w[2], all;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    place[i] = i0 + i >= 0 && i0 + i < v.V ? place_of(key_of((float)v.row[i0 + i]), i0 + i) : 0;
    const double rel = wt.rel(key_at(place[i]));
    w[i] = place[i] != 0 && place[i] >= cut && rel >= s.min_p ? wt.fix(rel) : 0;
  }
  at += block_before64<kRowWaves>(w[0] + w[1], s_sum, &all);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (at <= target && at + w[i] > target) draw(place[i], total);
    at += w[i];
  }
}

// One workgroup a row, bound by the latency of its steps, loads and barriers in turn: 12 us for one row of 151936
// with top-k 50 and top-p, 50 for 512 of them or of mixed settings, two workgroups a CU.
template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(Staged p) {
  __shared__ u64 s_list[kList], s_w[kList], s_sub[kSubsMost], s_sum[kRowWaves], s_out[6];
  __shared__ double s_powers[kPowers];
  __shared__ int s_n, s_m;
  const SampleParams& a = p.a;
  const int64_t q = blockIdx.x, r = p.r0 + q;
  // what any kind of row may need goes out together (a row of another kind leaves it unread)
  constexpr int kPerGroup = kGroups / kRowThreads;
  const int groups = (int)(((int64_t)p.n_sub * kSub) >> p.gshift), j0 = 2 * threadIdx.x;
  uint32_t g[kPerGroup];
#pragma unroll
  for (int i = 0; i < kPerGroup; ++i) {
    const int at = threadIdx.x + i * kRowThreads;
    g[i] = p.may_k && at < groups ? p.group[q * kGroups + at] : 0;
  }
  u64 sub[2], crossing[kCross];
#pragma unroll
  for (int i = 0; i < 2; ++i) sub[i] = p.may_sum && j0 + i < p.n_sub ? p.sums[q * p.n_sub + j0 + i] : 0;
#pragma unroll
  for (int i = 0; i < kCross; ++i) crossing[i] = p.may_p ? p.crossing[q * kCross + i] : 0;
  const int n_list = p.may_p ? p.n_list[q] : 0;
  const u64 list0 = p.may_p ? p.list[q * kList + threadIdx.x] : 0;
  const RowSettings s = settings_of(a, r);
  const u64 first = row_first(p, q);
  if (settled(a, r, s, first)) return;
  fill_powers(s_powers);
  const RowKind kind = kind_of(s, a.V);
  const RowView<T> v(a, r);
  const Weigh wt = weigh_of(a, s, key_at(first), s_powers);

  int n = 0;  // list entries
  if (kind == kTopKRow) {
    // A key that at least k groups reach: a histogram of the groups' distances below the largest key; the bin of the
    // k-th from the top by one wave (32 bins a lane, read in an order that meets every LDS bank).
    uint32_t* const s_cnt = reinterpret_cast<uint32_t*>(s_list);
    for (int i = threadIdx.x; i < kBins; i += kRowThreads) s_cnt[i] = 0;
    if (threadIdx.x == 0) s_n = s_m = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPerGroup; ++i)
      if (g[i] != 0) {
        atomicAdd(&s_cnt[distance_bin(wt.key_m - g[i])], 1u);
      }
    __syncthreads();
    if (wave_id() == 0) {
      const int lane = lane_id(), b0 = 32 * lane;
      uint32_t sum = 0;
#pragma unroll 8
      for (int i = 0; i < 32; ++i) sum += s_cnt[b0 + ((i + lane) & 31)];
      const uint32_t to = (uint32_t)wave_scan64(sum, Sum64());
      uint32_t at = to - sum;
      if (lane == 63 && to < s.k) s_out[0] = kBins;
      if (at < s.k && to >= s.k) {
        int b = b0;
        while (at + s_cnt[b] < s.k) at += s_cnt[b++];
        s_out[0] = b;
      }
    }
    __syncthreads();
    // d is below the bin's upper edge
    const uint32_t bin = (uint32_t)s_out[0];
    const float edge = __uint_as_float((bin + 1 + kOneBits) << 17);
    const uint32_t bound = bin < kBins && edge < (float)wt.key_m ? wt.key_m - (uint32_t)edge : 1;
    // the groups that reach it, then their tokens
    int* const s_group = reinterpret_cast<int*>(s_w);
    {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kPerGroup; ++i) c += g[i] >= bound;
      int at = append(&s_m, c);
#pragma unroll
      for (int i = 0; i < kPerGroup; ++i)
        if (g[i] >= bound) s_group[at++] = threadIdx.x + i * kRowThreads;
    }
    __syncthreads();
    const int n_group = s_m, lanes = 1 << (p.gshift - 3), per = kRowThreads / lanes;
    for (int first_i = 0; first_i < n_group; first_i += 4 * per) {
      const int i0 = first_i + threadIdx.x / lanes;
      Chunk<T> c[4];
      int64_t at0[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = i0 + j * per;
        at0[j] = ((int64_t)(i < n_group ? s_group[i] : 0) << p.gshift) - v.lead + (threadIdx.x % lanes) * kWaveLoad;
        c[j] = load_chunk(v, at0[j]);
      }
      uint32_t hits = 0;  // a bit for each that reaches the bound; they are few
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float l[kWaveLoad];
        chunk_logits(v, at0[j], c[j], l);
#pragma unroll
        for (int u = 0; u < kWaveLoad; ++u)
          hits |= i0 + j * per < n_group && key_of(l[u]) >= bound ? 1u << (j * kWaveLoad + u) : 0u;
      }
      int at = append(&s_n, __popc(hits));
      for (; hits != 0; hits &= hits - 1, ++at) {
        const int b = __ffs((int)hits) - 1, j = b / kWaveLoad;
        const int64_t i = (j == 0 ? at0[0] : j == 1 ? at0[1] : j == 2 ? at0[2] : at0[3]) + b % kWaveLoad;
        if (at < kList) s_list[at] = place_of(key_of((float)v.row[i]), i);
      }
    }
    __syncthreads();
    n = s_n;
  } else if (kind == kTopPRow) {
    n = n_list;
    if ((int)threadIdx.x < n) s_list[threadIdx.x] = list0;
    for (int i = threadIdx.x + kRowThreads; i < n && i < kList; i += kRowThreads) s_list[i] = p.list[q * kList + i];
  }
  __syncthreads();
  if (kind == kWholeRow || n > kList) {
    sample_row<T>(a, r, s, wt, RowShared{s_sum, s_out, s_w, reinterpret_cast<uint32_t*>(s_list)});
    return;
  }

  draw_row(a, r, s, v, wt, kind, n, p.n_sub, sub, crossing, FinishShared{s_list, s_w, s_sub, s_sum, s_out, &s_n, &s_m});
}

// ---------------------------------------------------------------- a short row
// Up to kRowMost logits, in one launch: the row, read once, is the list.  A radix descent reads it up to 8 times from
// L1, between barriers: 64 rows of 4096 with top-k and top-p took 35 us, so 20.  Without either there is no cut to find,
// and the two passes of sample_row over the cached row are the shorter way (10 us; by the list 43).
template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_short_kernel(SampleParams a) {
  __shared__ u64 s_list[kList], s_w[kList], s_sub[4], s_sum[kRowWaves], s_out[6];
  __shared__ double s_powers[kPowers];
  __shared__ int s_n, s_m;
  const int64_t r = blockIdx.x;
  const RowView<T> v(a, r);
  const int lead = v.lead % kLoad;
  uint32_t key[2][kLoad];  // (a row that begins between two borders takes one load more than kRowMost / kTile)
  int64_t i0[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    i0[j] = ((int64_t)j * kRowThreads + threadIdx.x) * kLoad - lead;
    if (j == 0 || i0[j] < a.V)
      load_keys(v.row, i0[j], v.V, key[j]);
    else
#pragma unroll
      for (int u = 0; u < kLoad; ++u) key[j][u] = 0;
  }
  const RowSettings s = settings_of(a, r);
  fill_powers(s_powers);
  if (threadIdx.x == 0) s_n = s_m = 0;
  u64 first = 0;
  int c = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int u = 0; u < kLoad; ++u) {
      const u64 x = place_of(key[j][u], i0[j] + u);
      first = x > first ? x : first;
      c += x != 0;
    }
  first = wave_max64(first);
  if (lane_id() == 0) s_sum[wave_id()] = first;
  __syncthreads();
#pragma unroll 4
  for (int j = 0; j < kRowWaves; ++j) first = s_sum[j] > first ? s_sum[j] : first;
  if (settled(a, r, s, first)) return;
  const Weigh wt = weigh_of(a, s, key_at(first), s_powers);
  if (s.k >= a.V && !(s.p < 1)) {
    sample_row<T>(a, r, s, wt, RowShared{s_sum, s_out, s_w, reinterpret_cast<uint32_t*>(s_list)});
    return;
  }
  int at = append(&s_n, c);
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int u = 0; u < kLoad; ++u)
      if (key[j][u] != 0) s_list[at++] = place_of(key[j][u], i0[j] + u);
  __syncthreads();
  const int n = s_n;
  __syncthreads();
  u64 sub[2] = {0, 0};
  const u64 crossing[kCross] = {0, 0, 0};
  draw_row(a, r, s, v, wt, kTopKRow, n, (int)((v.V + v.lead + kSub - 1) / kSub), sub, crossing,
           FinishShared{s_list, s_w, s_sub, s_sum, s_out, &s_n, &s_m});
}

// Rows of one launch: their workspace (up to 85 KB each) stays under 180 MB.
constexpr int64_t kRowsMost = 2048;

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

bool is_staged(int64_t V) { return V > kRowMost && V <= kStagedMost; }

int subs_of(int64_t V) { return (int)((V + kWaveLoad - 1 + kSub - 1) / kSub); }

struct StagedSizes {
  size_t first, group, hist, list, n_list, sums, crossing;
  size_t all() const { return first + group + hist + list + n_list + sums + crossing; }
};
StagedSizes staged_sizes(int64_t R, int64_t V) {
  const size_t rows = (size_t)(R < kRowsMost ? R : kRowsMost), subs = (size_t)subs_of(V);
  return {align256(rows * subs * 8), align256(rows * kGroups * 4), align256(rows * kBins * 8), align256(rows * kList * 8),
          align256(rows * 4), align256(rows * subs * 8), align256(rows * kCross * 8)};
}

template <class T>
hipError_t run_staged(const SampleParams& a, char* ws, hipStream_t stream) {
  Staged p{};
  p.a = a;
  p.n_sub = subs_of(a.V);
  // A sub-block per wave.  With 2, 4 and 9 each, 512 rows of 151936 with settings of their own take the three launches
  // 181, 206 and 269 us, so 151: a launch passes over many rows, and the others need workgroups enough for every CU.
  p.n_seg = (p.n_sub + 3) / 4;
  p.gshift = 3;
  while (((int64_t)p.n_sub * kSub) >> p.gshift > kGroups) ++p.gshift;
  const StagedSizes z = staged_sizes(a.R, a.V);
  p.first = reinterpret_cast<u64*>(ws);
  p.group = reinterpret_cast<uint32_t*>(ws += z.first);
  p.hist = reinterpret_cast<u64*>(ws += z.group);
  p.list = reinterpret_cast<u64*>(ws += z.hist);
  p.n_list = reinterpret_cast<int*>(ws += z.list);
  p.sums = reinterpret_cast<u64*>(ws += z.n_list);
  p.crossing = reinterpret_cast<u64*>(ws += z.sums);
  // rows' kinds, as far as the host knows them
  const bool greedy = !a.tau_rows && !(a.tau > 0);
  const bool all_k = !a.k_rows && a.k > 0 && a.k < a.V;
  p.may_k = !greedy && (a.k_rows || (all_k && a.k <= kTopK));
  p.may_p = !greedy && !all_k && (a.p_rows || a.p < 1);
  p.may_sum = !greedy && !all_k;
  for (p.r0 = 0; p.r0 < a.R; p.r0 += kRowsMost) {
    const int64_t rows = a.R - p.r0 < kRowsMost ? a.R - p.r0 : kRowsMost;
    const unsigned blocks = (unsigned)(rows * p.n_seg);
    sample_max_kernel<T><<<blocks, 256, 0, stream>>>(p);
    if (p.may_p) {
      const unsigned wide = (unsigned)(rows * ((p.n_sub + kHistWaves - 1) / kHistWaves));
      sample_hist_kernel<T><<<wide, 64 * kHistWaves, 0, stream>>>(p);
    }
    if (p.may_sum) sample_sums_kernel<T><<<blocks, 256, 0, stream>>>(p);
    sample_finish_kernel<T><<<(unsigned)rows, kRowThreads, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// The call without its first r0 rows.
template <class T>
SampleParams rows_from(SampleParams a, int64_t r0) {
  auto from = [&](const float*& x) { x = x ? x + r0 : x; };
  a.R -= r0;
  a.logits = static_cast<const T*>(a.logits) + r0 * a.ld;
  a.u = static_cast<const char*>(a.u) + r0 * (a.u64 ? 8 : 4);
  from(a.tau_rows);
  from(a.p_rows);
  from(a.min_p_rows);
  a.k_rows = a.k_rows ? a.k_rows + r0 : a.k_rows;
  a.token += r0;
  a.logprob += r0;
  return a;
}

template <class T>
hipError_t run(const SampleParams& a, char* ws, hipStream_t stream) {
  if (is_staged(a.V)) return run_staged<T>(a, ws, stream);
  constexpr int64_t kMost = 1 << 21;  // rows: a grid has fewer than 2^32 threads
  for (int64_t r0 = 0; r0 < a.R; r0 += kMost) {
    const SampleParams p = rows_from<T>(a, r0);
    const unsigned rows = (unsigned)(p.R < kMost ? p.R : kMost);
    if (a.V <= kRowMost)
      sample_short_kernel<T><<<rows, kRowThreads, 0, stream>>>(p);
    else
      sample_row_kernel<T><<<rows, kRowThreads, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

size_t sample_workspace_bytes(int64_t R, int64_t V) { return is_staged(V) ? staged_sizes(R, V).all() : 0; }

hipError_t sample_launch(int dtype, SampleParams p, char* ws, hipStream_t stream) {
  if (p.R == 0) return hipSuccess;
  int bits = 0;
  while (bits < 31 && ((int64_t)1 << bits) < p.V) ++bits;
  p.one = (double)((int64_t)1 << (bits < 12 ? 50 : 62 - bits));
  hipError_t e = hipSuccess;
  timing_begin(kKindSample, stream);
  switch (dtype) {
    case kBF16: e = run<bf16_t>(p, ws, stream); break;
    case kF16: e = run<f16_t>(p, ws, stream); break;
    case kF32: e = run<float>(p, ws, stream); break;
    default: return hipErrorInvalidValue;
  }
  timing_end(kKindSample, stream);
  return e;
}

}  // namespace swvr
