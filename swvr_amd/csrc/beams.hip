// Beam search's step (no counterpart in the reference): the best continuations of each sequence over its beams and the
// vocabulary, and the beams' states taken along.
//
// Selection.  With lse[w] = log sum_v exp(l[w, v]) a candidate is (w, v) with sum scores[w] + l[w, v] - lse[w] and rank
// sum / length^alpha; the k of the largest rank are kept, equal ones by beam, then by logit, then by index.  Within a
// beam the ranks are in the order of the logits, so the arithmetic decides between beams alone; there candidates lie
// close together (256 ranked ones of a step are some 1e-3 apart), so sums are formed in fp64: an exponential is off by
// 1.1e-12 of itself and an lse by less, where fp32's 1e-7 would swap a pair in one of a few thousand steps.  What is
// summed in which order depends on V alone (row_sum): the same beams have the same sums wherever they stand.
//
// Launches:
//   beam_scan_kernel   reads the logits once: per group of 128 its maximum, per sub-block of 2048 (a wave) its own and
//                      the sum of exponentials relative to it;
//   beam_row_kernel    per beam the lse, and its own k best: they lie in the k groups of the largest maxima (equal ones
//                      by index), which alone are read again;
//   beam_merge_kernel  per sequence the best of its beams' lists;
// the last two in one, a workgroup per sequence (beam_pick_kernel), for up to 256 candidates.
#include <algorithm>

#include "common.hpp"
#include "launch.hpp"
#include "rows.hpp"

namespace swvr {

namespace {

constexpr int kGroup = 128, kLane = 8, kStep = 64 * kLane, kSteps = 4, kSub = kSteps * kStep, kSubGroups = kSub / kGroup;
constexpr int kScanWaves = 4, kGroupsMost = (int)(kBeamVocabMost / kGroup), kListMost = 4096;

struct BeamWork {
  BeamParams a;
  int n_sub, n_seg, n_group;
  float* group;      // [rows][n_group] maxima, n_group = kSubGroups n_sub
  float* sub_max;    // [rows][n_sub]
  double* sub_sum;   // [rows][n_sub]
  double* rank;      // [rows][k]
  double* sum;       // [rows][k]
  int* token;        // [rows][k]
  int* count;        // [rows]
  u64* part_key;     // [B][parts][k], of a merge in two launches
  uint16_t* part_from;
};

__device__ __forceinline__ double score_of(const BeamParams& a, int64_t row) {
  return a.s64 ? static_cast<const double*>(a.scores)[row] : (double)static_cast<const float*>(a.scores)[row];
}
// A beam whose score is -inf, +inf or NaN has no candidates.
__device__ __forceinline__ bool alive(double score) { return fabs(score) < __builtin_huge_val(); }

// 2^(n + f) in fp64 by the Chebyshev interpolant of degree 8 on [-1/2, 1/2], 1.1e-12 of itself off; n from -1022 on
// as kRound + n, whose low bits it is.
constexpr double kLog2e64 = 1.4426950408889634074, kRound = 6755399441055744.0;  // 1.5 2^52: sums with it are whole numbers
__device__ __forceinline__ double pow2(double f, double n) {
  double p = 1.3255224887502117e-06;
  p = fma(p, f, 1.531007940254368e-05);
  p = fma(p, f, 0.0001540345585240991);
  p = fma(p, f, 0.0013333450567999414);
  p = fma(p, f, 0.009618129159402628);
  p = fma(p, f, 0.05550410941205934);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805459335);
  p = fma(p, f, 1.0);
  // (on the high word alone: a 64-bit shift and addition are two instructions for one)
  return __hiloint2double(__double2hiint(p) + (__double2loint(n) << 20), __double2loint(p));
}
// e^(x - m), about 2^-1000 for what lies below, and for NaN.
__device__ __forceinline__ double exp_rel(float x, double m) {
  const double d = fmax((double)x - m, -693.0), y = fma(d, kLog2e64, kRound);
  return pow2(fma(d, kLog2e64, kRound - y), y);
}

template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)));
}
// Maximum over groups of 8 lanes (quad_perm 1 0 3 2, 2 3 0 1, row_half_mirror), and over the wave (x8: max8's).
__device__ __forceinline__ float max8(float x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  return dpp_max<0x141>(x);
}
__device__ __forceinline__ float max64(float x8) {
  x8 = dpp_max<0x140>(x8);  // row_mirror
  float m = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 0));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 16)));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 32)));
  return fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 48)));
}

struct AddF64 {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const {
    return (u64)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
  }
};
__device__ __forceinline__ double wave_sum_f64(double x) {
  return __longlong_as_double((long long)last_lane64(wave_scan64((u64)__double_as_longlong(x), AddF64())));
}

// The sum of a row's exponentials relative to m from its sub-blocks' by(i) = e^(max_i - m) and sum(i): lane l's l, l + 64,
// ... one after another, then over the wave.  The kernels that need it share this order, each wave with all of it.
template <class By, class Sum>
__device__ __forceinline__ double row_sum(int n_sub, By&& by, Sum&& sum) {
  double x = 0;
#pragma unroll 1
  for (int i = lane_id(); i < n_sub; i += 64) x = fma(sum(i), by(i), x);
  return wave_sum_f64(x);
}
// (0 for a sub-block without candidates)
__device__ __forceinline__ double sub_weight(float mi, float m) { return mi > kNegInf ? exp((double)mi - (double)m) : 0.0; }

// kLane consecutive logits from any element on (rows begin anywhere where V is odd), -inf past the row's end.
template <class T>
using Logits = typename Vec8<T>::type;
static_assert(kLane == 8, "a vector of 8 a lane");
template <class T>
__device__ __forceinline__ Logits<T> whole_logits(const T* x) {
  typedef Logits<T> __attribute__((aligned(sizeof(T)))) Unaligned;
  return *reinterpret_cast<const Unaligned*>(x);
}
template <class T>
__device__ __forceinline__ Logits<T> load_logits(const T* x, int64_t i, int64_t V) {
  if (i + kLane <= V) return whole_logits(x + i);
  Logits<T> c;
#pragma unroll
  for (int u = 0; u < kLane; ++u) c[u] = i + u < V ? x[i + u] : (T)kNegInf;
  return c;
}

// Bound by the vector units: 21.5 instructions for a logit of each lane, 12.7 of them fp64's, of 4 cycles each, keep them
// busy in 99% of the cycles in which a CU has waves and in 80% of all: 512 rows of 151936 in bf16 54 us, where reading them
// takes 32.  (A few rows are bound by the launch and one round trip, 5 us.)  A wave takes
// as many logits as it can have on the way at once, and a row is spread over many.
template <class T>
__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(BeamWork p) {
  const int64_t row = blockIdx.x / p.n_seg;
  const int sub = (int)(blockIdx.x % p.n_seg) * kScanWaves + wave_id();
  if (sub >= p.n_sub) return;
  if ((p.a.finished && p.a.finished[row]) || !alive(score_of(p.a, row))) return;
  const T* const x = static_cast<const T*>(p.a.logits) + row * p.a.ld;
  const int64_t i0 = (int64_t)sub * kSub + lane_id() * kLane, V = p.a.V;
  Logits<T> c[kSteps];
  if ((int64_t)(sub + 1) * kSub <= V) {  // (the whole wave's: all loads go out before the first is waited for)
#pragma unroll
    for (int j = 0; j < kSteps; ++j) c[j] = whole_logits(x + i0 + j * kStep);
  } else {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) c[j] = load_logits(x, i0 + j * kStep, V);
  }
  float m = kNegInf, mine = kNegInf;  // mine: of the group of 16 lanes in step lane % 16
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    float k = kNegInf;
#pragma unroll
    for (int u = 0; u < kLane; ++u) k = fmaxf(k, (float)c[j][u]);  // (NaN: the other)
    k = dpp_max<0x140>(max8(k));  // (row_mirror)
    mine = (lane_id() & 15) == j ? k : mine;
    m = fmaxf(m, k);
  }
  m = max64(m);
  const double by = m > kNegInf && m < kPosInf ? (double)m : 0.0;
  double sum = 0;
  if (fabsf(m) < 0x1p22f) {
    // Two operations less: powers of 2 relative to 2^M, M next to m log2 e, as xL - M - n in one fma is exact but for its
    // last rounding (L's own error is taken off again with 2^(M - mL)); and m - 693 in fp32 is within 1.
    const double M = rint(by * kLog2e64), base = kRound - M;
    const float low = m - 693.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int u = 0; u < kLane; ++u) {
        const double x = __builtin_amdgcn_fmed3f((float)c[j][u], low, m), y = fma(x, kLog2e64, base);  // (NaN: low)
        sum += pow2(fma(x, kLog2e64, base - y), y);
      }
    sum *= pow2(fma(-by, kLog2e64, M), kRound);
  } else {
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int u = 0; u < kLane; ++u) sum += exp_rel((float)c[j][u], by);
  }
  sum = wave_sum_f64(sum);
  static_assert(kGroup == 16 * kLane, "a group is 16 lanes' logits of a step");
  if ((lane_id() & 15) < kSteps)
    p.group[row * p.n_group + sub * kSubGroups + (lane_id() & 15) * 4 + lane_id() / 16] = mine;
  if (lane_id() == 0) {
    p.sub_max[row * p.n_sub + sub] = m;
    p.sub_sum[row * p.n_sub + sub] = sum;
  }
}

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// How many of s[0 .. n - 1] (n padded with zeros to a multiple of kPad) are larger than x.
constexpr int kPad = 8;
__device__ __forceinline__ int above(const u64* s, int n, u64 x) {
  int c = 0;
#pragma unroll 1
  for (int i = 0; i < n; i += kPad) {
#pragma unroll
    for (int u = 0; u < kPad; ++u) c += s[i + u] > x;
  }
  return c;
}

constexpr int kRowThreads = 256;

// What a candidate's sum is divided by (lengths of 0 count as 1).
__device__ __forceinline__ int64_t length_of(const BeamParams& a, int64_t row, int more) { return a.lengths[row] + more; }
__device__ __forceinline__ double divisor(const BeamParams& a, int64_t length) {
  return pow((double)(length > 1 ? length : 1), a.alpha);
}
__device__ __forceinline__ bool divides(const BeamParams& a) { return a.lengths && a.alpha != 0; }

// A workgroup per beam.  Bound by what follows upon each other: 16 beams of 151936, 64 candidates 17 us (a logit at a
// time and the bound from the threads' best in both rounds, 31), 256 beams and candidates 113 us, most of it the order
// of a thousand group maxima.
template <class T>
__global__ __launch_bounds__(kRowThreads) void beam_row_kernel(BeamWork p) {
  __shared__ __attribute__((aligned(16))) u64 s_best[kRowThreads], s_list[kListMost + kPad];
  __shared__ u64 s_order[kBeamsMost];
  __shared__ int s_group[kBeamsMost];
  __shared__ float s_max[kRowThreads / 64];
  __shared__ u64 s_bound;
  __shared__ int s_n, s_more;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, k = p.a.k;
  const double score = score_of(p.a, row);
  double* const rank = p.rank + row * k;
  double* const sums = p.sum + row * k;
  int* const tokens = p.token + row * k;
  if (!alive(score)) {
    if (t == 0) p.count[row] = 0;
    return;
  }
  if (p.a.finished && p.a.finished[row]) {
    if (t == 0) {
      rank[0] = divides(p.a) ? score / divisor(p.a, length_of(p.a, row, 0)) : score;
      sums[0] = score;
      tokens[0] = (int)p.a.end_id;
      p.count[row] = 1;
    }
    return;
  }
  // ---- lse
  const float* const group = p.group + row * p.n_group;
  float m = kNegInf;
  for (int i = t; i < p.n_sub; i += kRowThreads) m = fmaxf(m, p.sub_max[row * p.n_sub + i]);
  m = max64(max8(m));
  if (lane_id() == 0) s_max[wave_id()] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 64; ++i) m = fmaxf(m, s_max[i]);
  if (!(m > kNegInf && m < kPosInf)) {  // nothing to choose (at +inf: no sum is a number)
    if (t == 0) p.count[row] = 0;
    return;
  }
  // (the exponentials by all threads, added in `first`: the list's room is free until then)
  static_assert(2 * (kBeamVocabMost / kSub) <= kListMost, "a weight and a sum for each sub-block");
  for (int i = t; i < p.n_sub; i += kRowThreads) {
    s_list[2 * i] = (u64)__double_as_longlong(sub_weight(p.sub_max[row * p.n_sub + i], m));
    s_list[2 * i + 1] = (u64)__double_as_longlong(p.sub_sum[row * p.n_sub + i]);
  }
  double rest = 0;  // lse - m
  auto add_up = [&]() {
    auto held = [&](int i) { return __longlong_as_double((long long)s_list[i]); };
    rest = log(row_sum(p.n_sub, [&](int i) { return held(2 * i); }, [&](int i) { return held(2 * i + 1); }));
  };
  // The k first of what n blocks of 8 hold, in order, to s_order; how many.  load(i, at, from): block i, its first one at
  // index `at`, those before `from` another block's.  A bound that k of them reach (where `bound` is 0: the k-th of the
  // threads' best), the few that reach it, and of these the places.  then(): once before the list's room is written, after a
  // barrier (where `bound` is 0).
  auto first = [&](int n, u64 bound, auto&& load, auto&& then) -> int {
    // f(value, index) for this thread's, but for blocks whose largest is below `least`; several are read before the
    // first is used
    auto each = [&](float least, auto&& f) {
      constexpr int kAhead = 4;
#pragma unroll 1
      for (int i0 = t; i0 < n; i0 += kAhead * kRowThreads) {
        decltype(load(0, i0, i0)) x[kAhead];
        int at[kAhead], from[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = i0 + u * kRowThreads;
          x[u] = load(i < n ? i : n - 1, at[u], from[u]);
          if (i >= n) from[u] = at[u] + kLane;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          float v[kLane], top = kNegInf;
#pragma unroll
          for (int e = 0; e < kLane; ++e) {
            v[e] = at[u] + e >= from[u] ? (float)x[u][e] : kNegInf;
            top = fmaxf(top, v[e]);  // (NaN: the other)
          }
          if (!(top >= least && top > kNegInf)) continue;
#pragma unroll
          for (int e = 0; e < kLane; ++e) f(v[e], at[u] + e);
        }
      }
    };
    if (bound == 0) {
      float best = kNegInf;
      each(kNegInf, [&](float x, int) { best = fmaxf(best, x); });
      const u64 mine = place_of(key_of(best), t);
      __syncthreads();
      s_best[t] = mine;
      if (t == 0) s_bound = 0;
      then();
      __syncthreads();
      if (mine && above(s_best, kRowThreads, mine) == k - 1) s_bound = (u64)key_at(mine) << 32;
      __syncthreads();
      bound = s_bound;
    }
    auto collect = [&]() -> int {
      __syncthreads();
      if (t == 0) s_n = 0;
      __syncthreads();
      const float least = logit_of(key_at(bound));
      each(least, [&](float x, int i) {
        if (!(x >= least)) return;
        const u64 y = place_of(key_of(x), i);
        if (y == 0 || y < bound) return;
        const int to = atomicAdd(&s_n, 1);
        if (to < kListMost) s_list[to] = y;
      });
      __syncthreads();
      return s_n;
    };
    int found = collect();
    if (found > kListMost) {
      // Too many reach it (equal ones, or the largest with few threads).  A higher bound, 8 bits at a time, by how many
      // there are of each next byte: `need` of those with the bits so far are still to be had.
      int* const count = reinterpret_cast<int*>(s_best);
      int need = k;
      bound = 0;
#pragma unroll 1
      for (int shift = 56; found > kListMost; shift -= 8) {
        count[t] = 0;
        __syncthreads();
        each(kNegInf, [&](float x, int i) {
          const u64 y = place_of(key_of(x), i);
          if (y && (shift == 56 || (y ^ bound) >> (shift + 8) == 0)) atomicAdd(&count[y >> shift & 255], 1);
        });
        __syncthreads();
        int more = 0;
#pragma unroll 4
        for (int i = t + 1; i < 256; ++i) more += count[i];
        if (more < need && more + count[t] >= need) {  // (one thread's)
          s_bound = bound | (u64)t << shift;
          s_n = more;
          s_more = count[t];
        }
        __syncthreads();
        bound = s_bound;
        need -= s_n;
        found = k - need + s_more;  // how many reach it
        __syncthreads();
      }
      found = collect();
    }
    if (t < kPad) s_list[found + t] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = t; i < found; i += kRowThreads) {
      const u64 x = s_list[i];
      const int r = above(s_list, found, x);
      if (r < k) s_order[r] = x;
    }
    __syncthreads();
    return found < k ? found : k;
  };
  const int groups = first(p.n_group / kLane, 0, [&](int i, int& at, int& from) {
    at = from = i * kLane;
    return whole_logits(group + at);
  }, add_up);
  if (t < groups) s_group[t] = (int)index_at(s_order[t]);
  // k groups: each has one that reaches the last one's largest
  const u64 reached = groups == k ? (u64)key_at(s_order[k - 1]) << 32 : 0;
  __syncthreads();
  const T* const x = static_cast<const T*>(p.a.logits) + row * p.a.ld;
  const int V = (int)p.a.V;
  const int n2 = first(groups * (kGroup / kLane), reached, [&](int i, int& at, int& from) {
    from = s_group[i / (kGroup / kLane)] * kGroup + i % (kGroup / kLane) * kLane;
    at = min(from, max(V - kLane, 0));  // (at the row's end the last 8)
    return V < kLane ? load_logits(x, at, V) : whole_logits(x + at);
  }, [] {});
  const double by = divides(p.a) ? divisor(p.a, length_of(p.a, row, 1)) : 1.0;
  if (t < n2) {
    const u64 y = s_order[t];
    const double s = score + (((double)logit_of(key_at(y)) - (double)m) - rest);
    rank[t] = s / by;
    sums[t] = s;
    tokens[t] = (int)index_at(y);
  }
  if (t == 0) p.count[row] = n2;
}

// Lists are merged two by two in LDS: an entry's place in both is its own and the number in the other list that come
// before it (of equal ones the lower beam's), found by halving.  A workgroup takes `per` of a sequence's beams; where
// that leaves several lists, a second launch merges those.  16 lists of 64 6.5 us, 256 of 256 28 us in two launches.  (A
// wave that takes the best head k times: 25 and 130.)
constexpr int kMergeHeld = 4096, kMergeThreads = 1024;
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamWork p, int per, bool second) {
  __shared__ u64 s_key[2][kMergeHeld];        // larger for a larger rank; 0: none
  __shared__ uint16_t s_from[2][kMergeHeld];  // beam << 8 | place in its list
  const int W = p.a.W, k = p.a.k, t = threadIdx.x, threads = blockDim.x, parts = (W + per - 1) / per;
  const int64_t b = second ? blockIdx.x : blockIdx.x / parts;
  const int w0 = second ? 0 : (int)(blockIdx.x % parts) * per;
  int lists = second ? parts : min(per, W - w0);
  for (int e = t; e < lists * k; e += threads) {
    const int w = w0 + e / k, i = e % k;
    if (second) {
      s_key[0][e] = p.part_key[b * parts * k + e];
      s_from[0][e] = p.part_from[b * parts * k + e];
    } else {
      const u64 y = (u64)__double_as_longlong(p.rank[(b * W + w) * k + i] + 0.0);  // (-0 is 0)
      s_key[0][e] = i >= p.count[b * W + w] ? 0 : y >> 63 ? ~y : y | (u64)1 << 63;
      s_from[0][e] = (uint16_t)(w << 8 | i);
    }
  }
  __syncthreads();
  int in = 0, top = 1;
  while (2 * top <= k) top *= 2;
#pragma unroll 1
  for (; lists > 1; lists = (lists + 1) / 2, in ^= 1) {
#pragma unroll 1
    for (int e = t; e < lists * k; e += threads) {
      const int l = e / k;
      const u64 x = s_key[in][e];
      int to = e - l * k;
      if ((l ^ 1) < lists) {
        const u64* const other = s_key[in] + (l ^ 1) * k;
        int n = 0;
#pragma unroll 1
        for (int step = top; step > 0; step >>= 1) {
          if (n + step > k) continue;
          const u64 y = other[n + step - 1];
          n += y > x || (y == x && (l & 1)) ? step : 0;
        }
        to += n;
      }
      if (to < k) {
        s_key[in ^ 1][(l >> 1) * k + to] = x;
        s_from[in ^ 1][(l >> 1) * k + to] = s_from[in][e];
      }
    }
    __syncthreads();
  }
  for (int r = t; r < k; r += threads) {
    if (!second && parts > 1) {
      p.part_key[(int64_t)blockIdx.x * k + r] = s_key[in][r];
      p.part_from[(int64_t)blockIdx.x * k + r] = s_from[in][r];
      continue;
    }
    const bool any = s_key[in][r] != 0;
    const int w = s_from[in][r] >> 8;
    const int64_t to = b * k + r, from = (b * W + w) * k + (s_from[in][r] & 255);
    const double score = any ? p.sum[from] : -__builtin_huge_val();
    p.a.token[to] = any ? p.token[from] : -1;
    p.a.parent[to] = any ? w : -1;
    if (p.a.s64) static_cast<double*>(p.a.score)[to] = score;
    else static_cast<float*>(p.a.score)[to] = (float)score;
  }
}

// ---- both in one launch: a workgroup per sequence, a wave per beam
// Bound by the latency of what follows upon each other: what the scan left, the few groups' logits, and one barrier
// before the merge: 4 beams of 151936, 4 candidates 6.9 us, 64 sequences of 8 beams, 16 candidates 12.3.  Loops stay loops,
// with as little as can be: unrolled throughout this took 15 us for the 4 beams, most of it to fetch its own instructions.
constexpr int kPickBeams = 16, kPickMost = 32, kPickAll = 256, kPickList = 256;

// base + i as a scalar base and a 32-bit offset (not an address in two registers for each load in flight).
template <class T>
__device__ __forceinline__ const T* at_offset(const T* base, int i) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + (uint32_t)i * (uint32_t)sizeof(T));
}

// A list of a wave in LDS: the places of values that are at least `least` go to its end, but for -inf.  (Past kPickList
// they are counted, not kept.)
struct WaveList {
  u64* at;
  int n;
  __device__ __forceinline__ void add(float x, int i, float least) {
    const bool in = x >= least && x > kNegInf;
    const uint64_t hit = __ballot(in);
    if (hit == 0) return;
    const int to = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
    if (in && to < kPickList) at[to] = (u64)__float_as_uint(x) << 32 | (uint32_t)i;  // (in_order makes places of them)
    n += __popcll(hit);
  }
  __device__ __forceinline__ static u64 raw(u64 place) {
    return (u64)__float_as_uint(logit_of(key_at(place))) << 32 | (uint32_t)index_at(place);
  }
  // The k first of all, in rounds of maxima: best(x) is this lane's first entry after x.  For lists that overflow
  // (many large ones with few lanes, equal ones).
  template <class F>
  __device__ __forceinline__ void by_rounds(int k, F&& best) {
    u64 last = ~0ull;
#pragma unroll 1
    for (n = 0; n < k; ++n) {
      last = wave_max64(best(last));
      if (last == 0) break;
      if (lane_id() == 0) at[n] = raw(last);
    }
  }
  // f(entry, its place) for the k first.
  template <class F>
  __device__ __forceinline__ void in_order(int k, F&& f) {
    wave_fence();
#pragma unroll 1
    for (int i = lane_id(); i < n; i += 64)
      at[i] = place_of(key_of(__uint_as_float((uint32_t)(at[i] >> 32))), (uint32_t)at[i]);
    if (lane_id() < kPad) at[n + lane_id()] = 0;
    wave_fence();
#pragma unroll 1
    for (int i = lane_id(); i < n; i += 64) {
      const u64 x = at[i];
      const int r = above(at, n, x);
      if (r < k) f(x, r);
    }
    wave_fence();
  }
};

// A value that k of the lanes' x or more reach: the k-th largest among the maxima of 4 lanes (up to 8), 2 (up to 16) or
// one; -inf where there are fewer.  s: 64 words of LDS.
__device__ __forceinline__ float reached_by(float x, int k, float* s) {
  int cells = 64, cell = lane_id();
  if (k <= 16) x = dpp_max<0xB1>(x), cells = 32, cell >>= 1;
  if (k <= 8) x = dpp_max<0x4E>(x), cells = 16, cell >>= 1;
  s[cell] = x;
  wave_fence();
  int larger = 0;
  const float4* const q = reinterpret_cast<const float4*>(s);
#pragma unroll 1
  for (int i = 0; i < cells / 4; i += 4)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float4 y = q[i + u];
      larger += (y.x > x) + (y.y > x) + (y.z > x) + (y.w > x);
    }
  wave_fence();
  // the smallest of those that fewer than k exceed
  return -max64(max8(larger < k ? -x : kNegInf));
}

template <class T>
__global__ __launch_bounds__(64 * kPickBeams) void beam_pick_kernel(BeamWork p) {
  __shared__ __attribute__((aligned(16))) u64 s_lists[kPickBeams][kPickList + kPad];
  __shared__ u64 s_chosen[kPickBeams][kPickMost];
  // candidate i of beam w at w k + i
  __shared__ double s_rank[kPickAll], s_sum[kPickAll];
  __shared__ int64_t s_length[kPickBeams];
  __shared__ int s_token[kPickAll], s_before[kPickAll], s_count[kPickBeams];
  const int b = (int)blockIdx.x;
  const int lane = lane_id(), k = p.a.k, W = p.a.W;
  u64* const chosen = s_chosen[wave_id()];
  const int w = wave_id(), n_group = p.n_group, n_sub = p.n_sub;
  // the beam's candidates to s_sum, s_token, best first; how many
  auto choose = [&]() -> int {
    const int64_t row = (int64_t)b * W + w;
    const float* const group = p.group + row * n_group;
    const double* const sub_sum = p.sub_sum + row * n_sub;
    const float* const sub_max = p.sub_max + row * n_sub;
    // All that is needed of a row of up to 262144 goes out at once (a round trip takes 1000 cycles and more); what is
    // further on is read where it is used.
    constexpr int kHeld = 32;
    float g[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (j % 16 == 0 && j * 64 >= n_group) break;
      g[j] = *at_offset(group, min(j * 64 + lane, n_group - 1));
    }
    const float max0 = sub_max[min(lane, n_sub - 1)], max1 = sub_max[min(lane + 64, n_sub - 1)];
    const double sum0 = sub_sum[min(lane, n_sub - 1)], sum1 = sub_sum[min(lane + 64, n_sub - 1)];
    const double score = score_of(p.a, row);
    const bool done = p.a.finished && p.a.finished[row];
    if (divides(p.a) && lane == 0) s_length[w] = length_of(p.a, row, done ? 0 : 1);
    if (!alive(score)) return 0;
    if (done) {
      if (lane == 0) {
        s_sum[w * k] = score;
        s_token[w * k] = (int)p.a.end_id;
      }
      return 1;
    }
    float top = kNegInf;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (j % 16 == 0 && j * 64 >= n_group) break;
      g[j] = j * 64 + lane < n_group ? g[j] : kNegInf;
      top = fmaxf(top, g[j]);
    }
#pragma unroll 1
    for (int i = kHeld * 64 + lane; i < n_group; i += 64) top = fmaxf(top, group[i]);
    const float m = max64(max8(top));
    if (!(m > kNegInf && m < kPosInf)) return 0;  // nothing to choose (at +inf: no sum is a number)
    // ---- the k first groups: a bound that k of them reach (the k-th of the lanes' best), the few that reach it, in order
    WaveList list{s_lists[wave_id()], 0};
    float least = reached_by(top, k, reinterpret_cast<float*>(list.at));
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (j % 16 == 0 && j * 64 >= n_group) break;
      list.add(g[j], j * 64 + lane, least);
    }
#pragma unroll 1
    for (int i = kHeld * 64; i < n_group; i += 64)
      list.add(i + lane < n_group ? group[min(i + lane, n_group - 1)] : kNegInf, i + lane, least);
    if (list.n > kPickList)
      list.by_rounds(k, [&](u64 last) {
        u64 y = 0;
#pragma unroll 1
        for (int i = lane; i < n_group; i += 64) {
          const u64 x = place_of(key_of(group[i]), i);
          y = x < last && x > y ? x : y;
        }
        return y;
      });
    list.in_order(k, [&](u64 x, int r) { chosen[r] = x; });
    // ---- the k first of their logits: none below the k-th group's largest
    const int groups = list.n < k ? list.n : k;
    least = groups == k ? logit_of(key_at(chosen[k - 1])) : kNegInf;
    const T* const x = static_cast<const T*>(p.a.logits) + row * p.a.ld;
    const int V = (int)p.a.V;
    // A lane's two of a group; at the row's end its last two are read, of which those from the lane's first on count.
    typedef T Pair __attribute__((ext_vector_type(2), aligned(sizeof(T))));
    static_assert(kGroup == 128, "two logits a lane");
    list.n = 0;
    constexpr int kAhead = 8;
#pragma unroll 1
    for (int s0 = 0; s0 < groups; s0 += kAhead) {
      Pair c[kAhead];
      int at[kAhead];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        at[s] = (int)index_at(chosen[min(s0 + s, groups - 1)]) * kGroup + lane * 2;
        c[s] = *reinterpret_cast<const Pair*>(at_offset(x, min(at[s], V - 2)));
      }
#pragma unroll
      for (int s = 0; s < kAhead; ++s) {
        if (s0 + s >= groups) break;
        const int from = min(at[s], V - 2);
        list.add(from == at[s] ? (float)c[s][0] : kNegInf, from, least);
        list.add(from + 1 >= at[s] ? (float)c[s][1] : kNegInf, from + 1, least);
      }
    }
    if (list.n > kPickList)
      list.by_rounds(k, [&](u64 last) {
        u64 y = 0;
#pragma unroll 1
        for (int s = 0; s < groups; ++s)
#pragma unroll 1
          for (int u = lane; u < kGroup; u += 64) {
            const int i = (int)index_at(chosen[s]) * kGroup + u;
            const u64 z = i < V ? place_of(key_of((float)x[i]), i) : 0;
            y = z < last && z > y ? z : y;
          }
        return y;
      });
    const double rest = log(row_sum(  // lse - m
        n_sub, [&](int i) { return sub_weight(i == lane ? max0 : i == lane + 64 ? max1 : sub_max[i], m); },
        [&](int i) { return i == lane ? sum0 : i == lane + 64 ? sum1 : sub_sum[i]; }));
    list.in_order(k, [&](u64 z, int r) {
      const double y = score + (((double)logit_of(key_at(z)) - (double)m) - rest);
      s_sum[w * k + r] = y;
      s_token[w * k + r] = (int)index_at(z);
    });
    return list.n < k ? list.n : k;
  };
  const int mine_n = choose();
  if (lane == 0) s_count[w] = mine_n;
  wave_fence();
  if (lane < k) {
    const double by = divides(p.a) ? divisor(p.a, s_length[w]) : 1.0;
    s_rank[w * k + lane] = lane < mine_n ? s_sum[w * k + lane] / by : -__builtin_huge_val();  // (none: after all that are)
    s_before[w * k + lane] = 0;
  }
  __syncthreads();
  // ---- how many come before each candidate of the wave's beam: 2^n lanes each, every one with its share of the others
  auto put = [&](int64_t at, int64_t token, int64_t parent, double score) {
    p.a.token[at] = token;
    p.a.parent[at] = parent;
    if (p.a.s64) static_cast<double*>(p.a.score)[at] = score;
    else static_cast<float*>(p.a.score)[at] = (float)score;
  };
  int width = 1;
  while (width < k) width *= 2;
  const int i = lane & (width - 1), share = lane / width, shares = 64 / width, all = W * k;
  const int me = w * k + i;
  const double mine = i < mine_n ? s_rank[me] : 0;
  int before = 0;
#pragma unroll 4
  for (int e = share; e < all; e += shares) {
    const double x = s_rank[e];
    before += x > mine || (x == mine && e < me);
  }
  if (i < mine_n) atomicAdd(&s_before[me], before);
  wave_fence();
  if (lane < mine_n) {
    const int to = s_before[w * k + lane];
    if (to < k) put((int64_t)b * k + to, s_token[w * k + lane], w, s_sum[w * k + lane]);
  }
  if (w == 0) {
    const int found = (int)wave_sum64(lane < W ? s_count[lane] : 0);
    if (lane >= found && lane < k) put((int64_t)b * k + lane, -1, -1, -__builtin_huge_val());
  }
}

int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

int beams_a_part(int W, int k) { return std::min(W, kMergeHeld / k); }
static_assert(kBeamsMost * kBeamsMost <= kMergeHeld / kBeamsMost * kMergeHeld, "what the parts leave is one workgroup's");

struct BeamSizes {
  int n_sub, n_group;
  int64_t group, sub_max, sub_sum, rank, sum, token, count, part_key, part_from;
  int64_t all() const { return group + sub_max + sub_sum + rank + sum + token + count + part_key + part_from; }
};
BeamSizes beam_sizes(int64_t B, int W, int64_t V, int k) {
  const int64_t rows = B * W;
  BeamSizes z;
  z.n_sub = (int)((V + kSub - 1) / kSub);
  z.n_group = z.n_sub * kSubGroups;
  z.group = rows * z.n_group * 4;
  z.sub_max = up8(rows * z.n_sub * 4);
  z.sub_sum = rows * z.n_sub * 8;
  z.rank = z.sum = rows * k * 8;
  z.token = up8(rows * k * 4);
  z.count = up8(rows * 4);
  const int per = beams_a_part(W, k);
  const int64_t parts = per < W ? B * ((W + per - 1) / per) * k : 0;
  z.part_key = parts * 8;
  z.part_from = up8(parts * 2);
  return z;
}

template <class T>
hipError_t run(BeamWork p, hipStream_t stream) {
  const int64_t rows = p.a.B * p.a.W;
  beam_scan_kernel<T><<<(unsigned)(rows * p.n_seg), 64 * kScanWaves, 0, stream>>>(p);
  // In one launch up to 256 candidates of 16 beams, 32 each.  (Both launches, 151936 logits: 4 beams of 4 11.5 us, in two
  // 18.1; 8 of 16 16.5, 20.9; 8 of 32 23.7, 22.7; 16 of 16 23.1, 22.4; 16 of 32 38.3, 24.4: a wave has a beam's list to
  // itself, and each candidate looks at all others.)
  if (p.a.W <= kPickBeams && p.a.k <= kPickMost && p.a.W * p.a.k <= kPickAll && p.a.V >= 2) {
    beam_pick_kernel<T><<<(unsigned)p.a.B, 64 * p.a.W, 0, stream>>>(p);
  } else {
    beam_row_kernel<T><<<(unsigned)rows, kRowThreads, 0, stream>>>(p);
    const int per = beams_a_part(p.a.W, p.a.k), parts = (p.a.W + per - 1) / per;
    auto threads = [&](int lists) { return (unsigned)std::min(kMergeThreads, (lists * p.a.k + 63) / 64 * 64); };
    beam_merge_kernel<<<(unsigned)(p.a.B * parts), threads(per), 0, stream>>>(p, per, false);
    if (parts > 1) beam_merge_kernel<<<(unsigned)p.a.B, threads(parts), 0, stream>>>(p, per, true);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- states
// A thread owns one column of V bytes of a state's beams: it reads the k parents' values before it writes any, so in
// place no other thread's reads are in the way, and a beam that keeps its parent costs nothing.  Bound by memory: 16 caches
// of 16 x 8 beams, 8 heads of 1000 of 1280 x 128 in bf16, in place: 1140 us, 5.2 TB/s of what changes place.
template <class Vec, int K>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderParams p, int64_t step0, int64_t b0, int j0) {
  const int64_t cols = p.run / (int64_t)sizeof(Vec);  // of a run
  const int64_t c = (step0 + blockIdx.x) * 256 + threadIdx.x, b = b0 + blockIdx.y;
  if (c >= cols * p.n1 * p.n2) return;
  int64_t from = c * (int64_t)sizeof(Vec), to = from;
  if (p.n1 * p.n2 > 1) {  // (below 2^32 bytes a beam then)
    const uint32_t c1 = (uint32_t)c / (uint32_t)cols, x0 = (uint32_t)c - c1 * (uint32_t)cols;
    const uint32_t x2 = c1 / (uint32_t)p.n1, x1 = c1 - x2 * (uint32_t)p.n1;
    from = (int64_t)x0 * sizeof(Vec) + x1 * p.src_1 + x2 * p.src_2;
    to = (int64_t)x0 * sizeof(Vec) + x1 * p.dst_1 + x2 * p.dst_2;
  }
  const char* const src = p.src[blockIdx.z] + b * p.src_b + from;
  char* dst = p.dst[blockIdx.z] + b * p.dst_b + j0 * p.dst_w + to;
  const int64_t at = b * p.k + j0;
  int n = p.k - j0 < K ? p.k - j0 : K;
  Vec v[K];
  uint64_t keep = 0;  // beams that stay as they are
#pragma unroll
  for (int j = 0; j < K; ++j) {
    v[j] = Vec{};
    if (K > 32 && j % 8 == 0) sched_fence();  // (not all parents in registers at once)
    if (j >= n) continue;
    const int64_t w = p.id64 ? static_cast<const int64_t*>(p.parents)[at + j] : (int64_t)static_cast<const int*>(p.parents)[at + j];
    if (p.in_place && w == j)
      keep |= (uint64_t)1 << j;
    else if (w >= 0 && w < p.W)
      v[j] = *reinterpret_cast<const Vec*>(src + w * p.src_w);
  }
  if (K > 32) asm volatile("" : "+s"(n));  // (nor the first loop's comparisons)
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j >= n) continue;
    if (!(keep >> j & 1)) *reinterpret_cast<Vec*>(dst) = v[j];
    dst += p.dst_w;
  }
}

template <class Vec, int K>
hipError_t reorder_run(const ReorderParams& p, hipStream_t stream) {
  // (a grid has fewer than 2^32 threads, and 2^16 workgroups along y)
  constexpr int64_t kMost = (int64_t)1 << 17, kSequences = 32768;
  const int64_t cols = p.run / (int64_t)sizeof(Vec) * p.n1 * p.n2, steps = (cols + 255) / 256;
  for (int j0 = 0; j0 < p.k; j0 += K)
    for (int64_t step = 0; step < steps; step += kMost) {
      const int64_t x = steps - step < kMost ? steps - step : kMost;
      const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kSequences, (((int64_t)1 << 24) - 1) / (x * p.n)));
      for (int64_t b = 0; b < p.B; b += most)
        reorder_kernel<Vec, K><<<dim3((unsigned)x, (unsigned)std::min(most, p.B - b), (unsigned)p.n), 256, 0, stream>>>(p, step, b, j0);
    }
  return hipGetLastError();
}

}  // namespace

size_t beams_workspace_bytes(int64_t B, int W, int64_t V, int k) { return (size_t)beam_sizes(B, W, V, k).all(); }

hipError_t beams_launch(int dtype, const BeamParams& a, char* ws, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  const BeamSizes z = beam_sizes(a.B, a.W, a.V, a.k);
  BeamWork p{};
  p.a = a;
  p.n_sub = z.n_sub;
  p.n_seg = (z.n_sub + kScanWaves - 1) / kScanWaves;
  p.n_group = z.n_group;
  p.group = reinterpret_cast<float*>(ws);
  p.sub_sum = reinterpret_cast<double*>(ws += z.group);
  p.rank = reinterpret_cast<double*>(ws += z.sub_sum);
  p.sum = reinterpret_cast<double*>(ws += z.rank);
  p.token = reinterpret_cast<int*>(ws += z.sum);
  p.count = reinterpret_cast<int*>(ws += z.token);
  p.sub_max = reinterpret_cast<float*>(ws += z.count);
  p.part_key = reinterpret_cast<u64*>(ws += z.sub_max);
  p.part_from = reinterpret_cast<uint16_t*>(ws += z.part_key);
  hipError_t e;
  timing_begin(kKindBeams, stream);
  switch (dtype) {
    case kBF16: e = run<bf16_t>(p, stream); break;
    case kF16: e = run<f16_t>(p, stream); break;
    default: e = run<float>(p, stream); break;
  }
  timing_end(kKindBeams, stream);
  return e;
}

hipError_t reorder_launch(const ReorderParams& p, hipStream_t stream) {
  if (p.n == 0 || p.B == 0 || p.k == 0 || p.run == 0 || p.n1 == 0 || p.n2 == 0) return hipSuccess;
  // the widest piece that every address is a multiple of
  uint64_t bits = (uint64_t)p.run | (uint64_t)p.src_b | (uint64_t)p.src_w | (uint64_t)p.src_1 | (uint64_t)p.src_2 |
                  (uint64_t)p.dst_b | (uint64_t)p.dst_w | (uint64_t)p.dst_1 | (uint64_t)p.dst_2;
  for (int i = 0; i < p.n; ++i) bits |= reinterpret_cast<uint64_t>(p.src[i]) | reinterpret_cast<uint64_t>(p.dst[i]);
  // (a thread holds k of them, at most 256 bytes of registers.  1 GB of bf16 in place: 8 beams 4.8 TB/s, 16 4.5, 32 5.0, 64
  // 3.1; into new tensors 16 beams 4.5, 32 4.9, 64 3.2, 200 from 8 2.9)
  const int most = p.k <= 16 ? 16 : p.k <= 32 ? 8 : 4;
  int width = 1;
  while (width < most && bits % (2 * width) == 0) width *= 2;
  hipError_t e;
  timing_begin(kKindReorder, stream);
  auto by_k = [&](auto x) {
    typedef decltype(x) Vec;
    if (p.k <= 4) return reorder_run<Vec, 4>(p, stream);
    if (p.k <= 8) return reorder_run<Vec, 8>(p, stream);
    if (p.k <= 16) return reorder_run<Vec, 16>(p, stream);
    if constexpr (sizeof(Vec) <= 8)
      if (p.k <= 32) return reorder_run<Vec, 32>(p, stream);
    if constexpr (sizeof(Vec) <= 4) return reorder_run<Vec, 64>(p, stream);
    return hipErrorInvalidValue;
  };
  switch (width) {
    case 16: e = by_k(uint4{}); break;
    case 8: e = by_k(uint2{}); break;
    case 4: e = by_k(uint32_t{}); break;
    case 2: e = by_k(uint16_t{}); break;
    default: e = by_k(uint8_t{}); break;
  }
  timing_end(kKindReorder, stream);
  return e;
}

}  // namespace swvr
