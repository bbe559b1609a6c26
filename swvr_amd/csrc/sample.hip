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

// Logits i0 .. i0 + L - 1 of a row as keys (0 outside 0 .. V - 1), in one load (fp32: 16 bytes each).  A row may begin
// anywhere: i0 + lead is a multiple of L, lead the row's distance from a border of L elements.
template <class T, int L>
__device__ __forceinline__ void load_keys(const T* row, int64_t i0, int64_t V, uint32_t (&key)[L]) {
  if (i0 >= 0 && i0 + L <= V) {
    struct alignas(L * sizeof(T) < 16 ? L * sizeof(T) : 16) X {
      T v[L];
    };
    const X x = *reinterpret_cast<const X*>(row + i0);
#pragma unroll
    for (int u = 0; u < L; ++u) key[u] = key_of((float)x.v[u]);
  } else {
#pragma unroll
    for (int u = 0; u < L; ++u) key[u] = i0 + u >= 0 && i0 + u < V ? key_of((float)row[i0 + u]) : 0;
  }
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
  uint32_t key_m;
  __device__ __forceinline__ double rel(uint32_t key) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: sums with it are whole numbers, in the low bits
    const double t = ((double)logit_of(key) - m) * to_log2;
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
    // (t is NaN where the largest logit is infinite: tokens equal to it, or under an infinite tau)
    return key == key_m ? 1.0 : key != 0 && t > -1000 ? w : 0.0;
  }
  // w in units of 2^-shift, to nearest: below 2^52, so the sum's low bits are the whole number
  __device__ __forceinline__ u64 fix(double w) const {
    return (u64)__double_as_longlong(fma(w, one, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ u64 wave_sum64(u64 x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

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
  u64 y = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 z = __shfl_up(y, o);
    if (lane_id() >= o) y += z;
  }
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
__device__ __forceinline__ u64 wave_max64(u64 x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 y = __shfl_xor(x, o);
    x = y > x ? y : x;
  }
  return x;
}

__device__ __forceinline__ Weigh weigh_of(const SampleParams& a, const RowSettings& s, uint32_t key_m,
                                          const double* powers) {
  Weigh w;
  w.powers = powers;
  w.m = (double)logit_of(key_m);
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
//                        reach it are read again, and their tokens that do are sorted.  Without, the list is
//                        sorted for the cut inside its bin, and the sub-block that holds the drawn token read again.
// So a row is read once with top-k, twice with min-p or nothing, three times with top-p, and its logits never sorted.
// A list that would pass kList tokens, or kSegList from one workgroup (equal logits, a nearly flat row) leaves its row to sample_row, in the same
// launch, as does a k above kTopK.  Every sum is one of whole numbers, so its order does not matter.
constexpr int kSub = 2048, kGroups = 4096, kList = 4096, kSegList = 2048, kTopK = 1024;
constexpr int64_t kRowMost = 4096, kStagedMost = ((int64_t)1 << 21) - 8;  // (groups of at most a wave's 512)
constexpr int kSubsMost = (int)(((int64_t)1 << 21) / kSub);
constexpr int kWaveLoad = 8;

enum RowKind { kGreedy, kTopKRow, kTopPRow, kSumRow, kWholeRow };
__device__ __forceinline__ RowKind kind_of(const RowSettings& s, int64_t V) {
  return s.tau == 0 ? kGreedy : s.k < V ? (s.k <= kTopK ? kTopKRow : kWholeRow) : s.p < 1 ? kTopPRow : kSumRow;
}

struct Staged {
  SampleParams a;
  int64_t r0;       // first row of this launch
  int n_sub;        // sub-blocks of a row
  int gshift;       // log2 of a group's logits
  int n_seg;        // workgroups of 4 waves per row in the first three launches
  u64* first;       // [rows][n_sub] place_of the sub-block's first token in order
  uint32_t* group;  // [rows][kGroups] largest keys
  u64* hist;        // [rows][kBins] weights
  u64* list;        // [rows][kList] places
  int* n_list;      // [rows]
  u64* sums;        // [rows][n_sub]
  u64* crossing;    // [rows][2]: the bin in which the prefix ends, the weight before it
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

// f(sub-block, first index of the lane's kWaveLoad logits, keys) over the sub-blocks of this wave.
template <class T, class F, class G>
__device__ __forceinline__ void each_sub(const Staged& p, const RowView<T>& v, F&& f, G&& done) {
  constexpr int kSteps = kSub / (64 * kWaveLoad);
  for (int sub = (int)(blockIdx.x % p.n_seg) * 4 + wave_id(); sub < p.n_sub; sub += 4 * p.n_seg) {
    uint32_t key[kSteps][kWaveLoad];
    const int64_t i0 = (int64_t)sub * kSub - v.lead + lane_id() * kWaveLoad;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) load_keys(v.row, i0 + j * 64 * kWaveLoad, v.V, key[j]);
#pragma unroll
    for (int j = 0; j < kSteps; ++j) f(sub, j, i0 + j * 64 * kWaveLoad, key[j]);
    done(sub);
  }
}

// A row's first token in order, by each wave for itself.
__device__ __forceinline__ u64 row_first(const Staged& p, int64_t q) {
  u64 first = 0;
  for (int i = lane_id(); i < p.n_sub; i += 64) {
    const u64 x = p.first[q * p.n_sub + i];
    first = x > first ? x : first;
  }
  return wave_max64(first);
}

// Bin of a key: its distance below the largest in units of 46 log2-steps of weight / kBins (past that, weights are 0),
// in fp32: no smaller for a smaller logit.
__device__ __forceinline__ float bin_scale(const Weigh& w) { return (float)(w.to_log2 * (kBins / 46.0)); }
__device__ __forceinline__ int bin_of(uint32_t key, const Weigh& w, float scale) {
  const float x = ((float)w.m - logit_of(key)) * scale;
  return key == w.key_m ? 0 : x < kBins - 1 ? (int)x : kBins - 1;
}

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
  u64 first = 0;
  each_sub(
      p, RowView<T>(p.a, r),
      [&](int sub, int j, int64_t i0, const uint32_t(&key)[kWaveLoad]) {
        uint32_t k = 0;
        int at = 0;
#pragma unroll
        for (int u = 0; u < kWaveLoad; ++u)
          if (key[u] > k) {
            k = key[u];
            at = u;
          }
        const u64 x = place_of(k, i0 + at);
        first = x > first ? x : first;
        if (kind != kTopKRow) return;
        for (int o = 1; o < lanes; o <<= 1) {
          const uint32_t y = __shfl_xor(k, o);
          k = y > k ? y : k;
        }
        if ((lane_id() & (lanes - 1)) == 0)
          p.group[q * kGroups + (((int64_t)sub * kSub + j * 64 * kWaveLoad + lane_id() * kWaveLoad) >> p.gshift)] = k;
      },
      [&](int sub) {
        first = wave_max64(first);
        if (lane_id() == 0) p.first[q * p.n_sub + sub] = first;
        first = 0;
      });
}

template <class T>
__global__ __launch_bounds__(256) void sample_hist_kernel(Staged p) {
  __shared__ u64 s_hist[kBins];
  __shared__ double s_powers[kPowers];
  const int64_t q = blockIdx.x / p.n_seg, r = p.r0 + q;
  const RowSettings s = settings_of(p.a, r);
  const u64 first = row_first(p, q);
  if (kind_of(s, p.a.V) != kTopPRow || first == 0) return;
  fill_powers(s_powers);
  for (int i = threadIdx.x; i < kBins; i += 256) s_hist[i] = 0;
  __syncthreads();
  const Weigh wt = weigh_of(p.a, s, key_at(first), s_powers);
  const float scale = bin_scale(wt);
  each_sub(
      p, RowView<T>(p.a, r),
      [&](int, int, int64_t, const uint32_t(&key)[kWaveLoad]) {
#pragma unroll
        for (int u = 0; u < kWaveLoad; ++u) {
          const u64 w = wt.fix(wt.rel(key[u]));
          if (w) atomicAdd(&s_hist[bin_of(key[u], wt, scale)], w);
        }
      },
      [](int) {});
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (s_hist[i]) atomicAdd(&p.hist[q * kBins + i], s_hist[i]);
}

template <class T>
__global__ __launch_bounds__(256) void sample_sums_kernel(Staged p) {
  __shared__ u64 s_sum[4], s_cross[2], s_list[kSegList];
  __shared__ double s_powers[kPowers];
  __shared__ int s_n, s_at;
  const int64_t q = blockIdx.x / p.n_seg, r = p.r0 + q;
  const RowSettings s = settings_of(p.a, r);
  const RowKind kind = kind_of(s, p.a.V);
  const u64 first = row_first(p, q);
  if ((kind != kTopPRow && kind != kSumRow) || first == 0) return;
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
      }
      at += w[i];
    }
    __syncthreads();
    cross = (int)s_cross[0];
    if (blockIdx.x % p.n_seg == 0 && threadIdx.x < 2) p.crossing[q * 2 + threadIdx.x] = s_cross[threadIdx.x];
  }
  __syncthreads();
  const Weigh wt = weigh_of(p.a, s, key_at(first), s_powers);
  const float scale = bin_scale(wt);
  u64 sum = 0;
  each_sub(
      p, RowView<T>(p.a, r),
      [&](int, int, int64_t i0, const uint32_t(&key)[kWaveLoad]) {
#pragma unroll
        for (int u = 0; u < kWaveLoad; ++u) {
          const int b = bin_of(key[u], wt, scale);
          if (b < cross) {
            const double w = wt.rel(key[u]);
            sum += w >= s.min_p ? wt.fix(w) : 0;
          } else if (b == cross && key[u] != 0) {
            const int at = atomicAdd(&s_n, 1);
            if (at < kSegList) s_list[at] = place_of(key[u], i0 + u);
          }
        }
      },
      [&](int sub) {
        sum = wave_sum64(sum);
        if (lane_id() == 0) p.sums[q * p.n_sub + sub] = sum;
        sum = 0;
      });
  if (kind != kTopPRow) return;
  // the bin's tokens of this workgroup to the row's list, whose order does not matter
  __syncthreads();
  const int n = s_n;
  if (threadIdx.x == 0 && n > 0) s_at = atomicAdd(&p.n_list[q], n <= kSegList ? n : kList + 1);
  __syncthreads();
  for (int i = threadIdx.x; i < n && n <= kSegList; i += 256)
    if (s_at + i < kList) p.list[q * kList + s_at + i] = s_list[i];
}

// s[0 .. n2), n2 a power of two, into descending (or ascending) order by kRowThreads threads.  A wave's pairs of
// a step of up to 64 lie in 128 elements of its own.
template <bool DESC>
__device__ __forceinline__ void bitonic_sort(u64* s, int n2) {
  for (int k = 2; k <= n2; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 128 || (j == 64 && k > 128) || k == 2)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int t = threadIdx.x; t < n2 / 2; t += kRowThreads) {
        const int i = (t & ~(j - 1)) * 2 + (t & (j - 1));
        const u64 a = s[i], b = s[i + j];
        const bool up = ((i & k) == 0) != DESC;  // this pair ascending
        if ((a > b) == up) {
          s[i] = b;
          s[i + j] = a;
        }
      }
    }
  __syncthreads();
}

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_finish_kernel(Staged p) {
  __shared__ u64 s_list[kList], s_w[kList], s_sub[kSubsMost], s_sum[kRowWaves], s_out[4];
  __shared__ double s_powers[kPowers];
  __shared__ int s_n;
  const SampleParams& a = p.a;
  const int64_t q = blockIdx.x, r = p.r0 + q;
  const RowSettings s = settings_of(a, r);
  const u64 first = row_first(p, q);
  if (settled(a, r, s, first)) return;
  fill_powers(s_powers);
  const RowKind kind = kind_of(s, a.V);
  const RowView<T> v(a, r);
  const Weigh wt = weigh_of(a, s, key_at(first), s_powers);
  constexpr int kPer = kList / kRowThreads;  // list entries of a thread
  const int t0 = threadIdx.x * kPer;
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();

  int n = 0;  // list entries
  if (kind == kTopKRow) {
    // a key that at least k tokens reach, from its upper 22 bits
    uint32_t* const s_cnt = reinterpret_cast<uint32_t*>(s_list);
    const int groups = (int)(((int64_t)p.n_sub * kSub) >> p.gshift);
    uint32_t g[kGroups / kRowThreads];
#pragma unroll
    for (int i = 0; i < kGroups / kRowThreads; ++i) {
      const int at = threadIdx.x + i * kRowThreads;
      g[i] = at < groups ? p.group[q * kGroups + at] : 0;
    }
    uint32_t bound = 0, before = 0;
    bool found = true;
#pragma unroll 1
    for (int sh = 21; sh >= 10 && found; sh -= 11) {
      for (int i = threadIdx.x; i < kBins; i += kRowThreads) s_cnt[i] = 0;
      if (threadIdx.x == 0) s_out[0] = ~0ull;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kGroups / kRowThreads; ++i)
        if (g[i] != 0 && (sh == 21 || (g[i] >> 21) == (bound >> 21)))
          atomicAdd(&s_cnt[(g[i] >> sh) & (kBins - 1)], 1u);
      __syncthreads();
      const int b1 = kBins - 1 - 2 * (int)threadIdx.x;
      const uint32_t n1 = s_cnt[b1], n0 = s_cnt[b1 - 1];
      u64 all;
      const uint32_t at = before + (uint32_t)block_before64<kRowWaves>(n1 + n0, s_sum, &all);
      if (at < s.k && at + n1 >= s.k) {
        s_out[0] = b1;
        s_out[1] = at;
      } else if (at + n1 < s.k && at + n1 + n0 >= s.k) {
        s_out[0] = b1 - 1;
        s_out[1] = at + n1;
      }
      __syncthreads();
      found = s_out[0] != ~0ull;
      if (found) {
        bound |= (uint32_t)s_out[0] << sh;
        before = (uint32_t)s_out[1];
      }
      __syncthreads();
    }
    if (bound == 0) bound = 1;
    // the groups that reach it, then their tokens
    int* const s_group = reinterpret_cast<int*>(s_w);
#pragma unroll
    for (int i = 0; i < kGroups / kRowThreads; ++i)
      if (g[i] >= bound) s_group[atomicAdd(&s_n, 1)] = threadIdx.x + i * kRowThreads;
    __syncthreads();
    const int n_group = s_n;
    __syncthreads();
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    const int lanes = 1 << (p.gshift - 3), per = kRowThreads / lanes;
#pragma unroll 2
    for (int i = threadIdx.x / lanes; i < n_group; i += per) {
      const int64_t i0 = ((int64_t)s_group[i] << p.gshift) - v.lead + (threadIdx.x % lanes) * kWaveLoad;
      uint32_t key[kWaveLoad];
      load_keys(v.row, i0, v.V, key);
#pragma unroll
      for (int u = 0; u < kWaveLoad; ++u)
        if (key[u] >= bound) {
          const int at = atomicAdd(&s_n, 1);
          if (at < kList) s_list[at] = place_of(key[u], i0 + u);
        }
    }
    __syncthreads();
    n = s_n;
  } else if (kind == kTopPRow) {
    n = p.n_list[q];
    for (int i = threadIdx.x; i < n && i < kList; i += kRowThreads) s_list[i] = p.list[q * kList + i];
  }
  if (kind == kWholeRow || n > kList) {
    __syncthreads();
    sample_row<T>(a, r, s, wt, RowShared{s_sum, s_out, s_w, reinterpret_cast<uint32_t*>(s_list)});
    return;
  }

  u64 cut = 0, total = 0;  // the last token of the prefix (0: every token), the kept weight
  int kept = 0;            // entries of the list up to the last that is in the prefix and not below min_p
  if (n > 0) {
    const int n2 = pow2_at_least(n);
    __syncthreads();
    for (int i = n + threadIdx.x; i < n2; i += kRowThreads) s_list[i] = 0;
    bitonic_sort<true>(s_list, n2);
    u64 place[kPer], w[kPer], sum = 0, all;
    double rel[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = t0 + i < n && (kind != kTopKRow || t0 + i < s.k);
      place[i] = in ? s_list[t0 + i] : 0;
      rel[i] = in ? wt.rel(key_at(place[i])) : 0;
      sum += w[i] = wt.fix(rel[i]);
    }
    u64 at = block_before64<kRowWaves>(sum, s_sum, &all);
    double limit = s.p < 1 ? s.p * (double)all : kPosInf;
    if (kind == kTopPRow) {
      at += p.crossing[q * 2 + 1];
      u64 z = 0, x;
      for (int i = threadIdx.x; i < kBins; i += kRowThreads) z += p.hist[q * kBins + i];
      x = block_sum64<kRowWaves>(z, s_sum);
      limit = s.p * (double)x;
    }
    if (!(limit > 0)) limit = 0.5;
    u64 n_prefix = 0, kept_w = 0;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool prefix = place[i] != 0 && (double)at < limit;
      at += w[i];
      const bool keep = prefix && rel[i] >= s.min_p;
      n_prefix += prefix;
      if (keep) atomicMax(&s_n, t0 + i + 1);
      kept_w += keep ? w[i] : 0;
      if (kind == kTopKRow) s_w[t0 + i] = keep ? w[i] : 0;
      rel[i] = keep ? 1 : 0;
    }
    n_prefix = block_sum64<kRowWaves>(n_prefix, s_sum);
    total = block_sum64<kRowWaves>(kept_w, s_sum);
    kept = s_n;
    cut = s_list[n_prefix - 1];
    __syncthreads();
    if (kind == kTopKRow) {
      // the kept ones by index, each with its place in the order
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (t0 + i < pow2_at_least(kept))
          s_list[t0 + i] = t0 + i < kept ? (u64)index_at(place[i]) << 32 | (u64)(t0 + i) : ~0ull;
      bitonic_sort<false>(s_list, pow2_at_least(kept));
      const double uz = s.u * (double)total;
      const u64 target = uz < (double)(total - 1) ? (u64)uz : total - 1;
      u64 x[kPer];
      sum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum += x[i] = t0 + i < kept ? s_w[(uint32_t)s_list[t0 + i]] : 0;
      at = block_before64<kRowWaves>(sum, s_sum, &all);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (at <= target && at + x[i] > target) s_out[0] = s_list[t0 + i] >> 32;
        at += x[i];
      }
    } else {
      // their weights join their sub-blocks' sums
      for (int i = threadIdx.x; i < p.n_sub; i += kRowThreads) s_sub[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (rel[i] != 0 && w[i]) atomicAdd(&s_sub[(index_at(place[i]) + v.lead) / kSub], w[i]);
    }
  }
  if (kind != kTopKRow) {
    // the sub-block that holds the token, then its place there
    __syncthreads();
    const int j0 = 2 * threadIdx.x;
    u64 x[2], all;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      x[i] = j0 + i < p.n_sub ? p.sums[q * p.n_sub + j0 + i] + (n > 0 ? s_sub[j0 + i] : 0) : 0;
    u64 at = block_before64<kRowWaves>(x[0] + x[1], s_sum, &all);
    total = all;
    const double uz = s.u * (double)total;
    const u64 target = uz < (double)(total - 1) ? (u64)uz : total - 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (at <= target && at + x[i] > target) {
        s_out[1] = j0 + i;
        s_out[2] = at;
      }
      at += x[i];
    }
    __syncthreads();
    const int64_t i0 = (int64_t)s_out[1] * kSub - v.lead + 2 * threadIdx.x;
    at = s_out[2];
    u64 w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t key = i0 + i >= 0 && i0 + i < v.V ? key_of((float)v.row[i0 + i]) : 0;
      const u64 place = place_of(key, i0 + i);
      const double rel = wt.rel(key);
      w[i] = place != 0 && place >= cut && rel >= s.min_p ? wt.fix(rel) : 0;
    }
    at += block_before64<kRowWaves>(w[0] + w[1], s_sum, &all);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (at <= target && at + w[i] > target) s_out[0] = (u64)(i0 + i);
      at += w[i];
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t token = (int64_t)s_out[0];
    const uint32_t key = key_of((float)v.row[token]);
    const double rel = key == wt.key_m ? 0.0 : ((double)logit_of(key) - wt.m) / s.tau;
    a.token[r] = token;
    a.logprob[r] = (float)(rel - log((double)total / a.one));
  }
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
          align256(rows * 4), align256(rows * subs * 8), align256(rows * 16)};
}

template <class T>
hipError_t run_staged(const SampleParams& a, char* ws, hipStream_t stream) {
  Staged p{};
  p.a = a;
  p.n_sub = subs_of(a.V);
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
  const bool may_p = !greedy && !all_k && (a.p_rows || a.p < 1), may_sum = !greedy && !all_k;
  for (p.r0 = 0; p.r0 < a.R; p.r0 += kRowsMost) {
    const int64_t rows = a.R - p.r0 < kRowsMost ? a.R - p.r0 : kRowsMost;
    // about 1024 workgroups for all rows, a sub-block at least per wave
    const int64_t want = (1024 + rows - 1) / rows, most = (p.n_sub + 3) / 4;
    p.n_seg = (int)(want < most ? want : most);
    const unsigned blocks = (unsigned)(rows * p.n_seg);
    sample_max_kernel<T><<<blocks, 256, 0, stream>>>(p);
    if (may_p) sample_hist_kernel<T><<<blocks, 256, 0, stream>>>(p);
    if (may_sum) sample_sums_kernel<T><<<blocks, 256, 0, stream>>>(p);
    sample_finish_kernel<T><<<(unsigned)rows, kRowThreads, 0, stream>>>(p);
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
  const bool staged = is_staged(p.V);
  hipError_t e = hipSuccess;
  timing_begin(kKindSample, stream);
  switch (dtype) {
    case kBF16:
      if (staged) e = run_staged<bf16_t>(p, ws, stream);
      else sample_row_kernel<bf16_t><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p);
      break;
    case kF16:
      if (staged) e = run_staged<f16_t>(p, ws, stream);
      else sample_row_kernel<f16_t><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p);
      break;
    case kF32:
      if (staged) e = run_staged<float>(p, ws, stream);
      else sample_row_kernel<float><<<(unsigned)p.R, kRowThreads, 0, stream>>>(p);
      break;
    default: return hipErrorInvalidValue;
  }
  timing_end(kKindSample, stream);
  return e != hipSuccess ? e : hipGetLastError();
}

}  // namespace swvr
