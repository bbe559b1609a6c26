// Beam search's step (no counterpart in the reference): the best continuations of each sequence over its beams and the
// vocabulary, and the beams' states taken along.
//
// Selection.  With lse[w] = log sum_v exp(l[w, v]) a candidate is (w, v) with sum scores[w] + l[w, v] - lse[w] and rank
// sum / length^alpha; the k of the largest rank are kept, equal ones by beam, then by logit, then by index.  Within a
// beam the ranks are in the order of the logits, so the arithmetic decides between beams alone; there candidates lie
// close together (256 ranked ones of a step are some 1e-3 apart), so sums are formed in fp64: an exponential is off by
// 1.1e-12 of itself and an lse by less, where fp32's 1e-7 would swap a pair in one of a few thousand steps.  What is
// summed in which order depends on V alone: the same beams have the same sums wherever they stand.
//
// Three launches:
//   beam_scan_kernel   reads the logits once: per sub-block of kSub (a wave) the maximum and the sum of exponentials
//                      relative to it, per group of 64 or 512 consecutive logits its maximum;
//   beam_row_kernel    per beam the lse, and its own k best: they lie in the k groups of the largest maxima (equal ones
//                      by index), which alone are read again;
//   beam_merge_kernel  per sequence the best of its beams' lists.
#include <algorithm>

#include "common.hpp"
#include "launch.hpp"
#include "rows.hpp"

namespace swvr {

namespace {

constexpr int kSub = 2048, kLane = 8, kSteps = kSub / (64 * kLane);
constexpr int kScanWaves = 4, kGroupsMost = 4096, kListMost = 4096;
constexpr int64_t kSmallGroups = (int64_t)kGroupsMost * 64;  // V up to which groups have 64 logits

struct BeamWork {
  BeamParams a;
  int n_sub, n_seg, gshift, n_group;
  float* sub_max;    // [rows][n_sub]
  double* sub_sum;   // [rows][n_sub]
  float* group;      // [rows][n_group]
  double* rank;      // [rows][k]
  double* sum;       // [rows][k]
  int* token;        // [rows][k]
  int* count;        // [rows]
};

__device__ __forceinline__ double score_of(const BeamParams& a, int64_t row) {
  return a.s64 ? static_cast<const double*>(a.scores)[row] : (double)static_cast<const float*>(a.scores)[row];
}
// A beam whose score is -inf, +inf or NaN has no candidates.
__device__ __forceinline__ bool alive(double score) { return fabs(score) < __builtin_huge_val(); }

// e^(x - m) in fp64: with t = (x - m) log2 e, n the whole number next to it, 2^n times 2^(t - n) by its Chebyshev
// interpolant of degree 8 on [-1/2, 1/2], 1.1e-12 of itself off.  About 2^-1000 for what lies below, and for NaN.
__device__ __forceinline__ double exp_rel(float x, double m) {
  constexpr double kLog2e64 = 1.4426950408889634074;
  constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: sums with it are whole numbers, in the low bits
  const double d = fmax((double)x - m, -693.0);
  const double y = fma(d, kLog2e64, kRound);
  const double f = fma(d, kLog2e64, kRound - y);
  double p = 1.3255224887502117e-06;
  p = fma(p, f, 1.531007940254368e-05);
  p = fma(p, f, 0.0001540345585240991);
  p = fma(p, f, 0.0013333450567999414);
  p = fma(p, f, 0.009618129159402628);
  p = fma(p, f, 0.05550410941205934);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805459335);
  p = fma(p, f, 1.0);
  return __longlong_as_double(__double_as_longlong(p) + ((long long)(int)__double_as_longlong(y) << 52));
}

template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true)));
}
// Maximum over groups of 8 lanes (quad_perm 1 0 3 2, 2 3 0 1, row_half_mirror), and over the wave.
__device__ __forceinline__ float max8(float x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  return dpp_max<0x141>(x);
}
__device__ __forceinline__ float max64(float x8) {  // x8: max8's
  x8 = dpp_max<0x140>(x8);  // row_mirror
  float m = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 0));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 16)));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 32)));
  return fmaxf(m, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x8), 48)));
}

// kLane consecutive logits from any element on (rows begin anywhere where V is odd).
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) LaneLogits {
  T v[kLane];
};

template <class T>
__global__ __launch_bounds__(64 * kScanWaves) void beam_scan_kernel(BeamWork p) {
  const int64_t row = blockIdx.x / p.n_seg;
  const int sub = (int)(blockIdx.x % p.n_seg) * kScanWaves + wave_id();
  if (sub >= p.n_sub) return;
  if ((p.a.finished && p.a.finished[row]) || !alive(score_of(p.a, row))) return;
  const T* const x = static_cast<const T*>(p.a.logits) + row * p.a.ld;
  const int64_t i0 = (int64_t)sub * kSub + lane_id() * kLane, V = p.a.V;
  float l[kSteps][kLane];
  LaneLogits<T> c[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; ++j)
    if (i0 + j * 64 * kLane + kLane <= V) c[j] = *reinterpret_cast<const LaneLogits<T>*>(x + i0 + j * 64 * kLane);
  float m = kNegInf;
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const int64_t i = i0 + j * 64 * kLane;
    if (i + kLane <= V) {
#pragma unroll
      for (int u = 0; u < kLane; ++u) l[j][u] = (float)c[j].v[u];
    } else {
#pragma unroll
      for (int u = 0; u < kLane; ++u) l[j][u] = i + u < V ? (float)x[i + u] : kNegInf;
    }
    float k = kNegInf;
#pragma unroll
    for (int u = 0; u < kLane; ++u) k = fmaxf(k, l[j][u]);  // (NaN: the other)
    k = max8(k);
    const int64_t g = (i0 - lane_id() * kLane + j * 64 * kLane) >> 6;  // first group of 64 of this step
    if (p.gshift == 6) {
      if ((lane_id() & 7) == 0 && g + lane_id() / 8 < p.n_group) p.group[row * p.n_group + g + lane_id() / 8] = k;
      m = fmaxf(m, k);
    } else {
      const float k64 = max64(k);
      if (lane_id() == 0 && (g >> 3) < p.n_group) p.group[row * p.n_group + (g >> 3)] = k64;
      m = fmaxf(m, k64);
    }
  }
  m = max64(m);
  const double by = m > kNegInf && m < kPosInf ? (double)m : 0.0;
  double sum = 0;
#pragma unroll
  for (int j = 0; j < kSteps; ++j)
#pragma unroll
    for (int u = 0; u < kLane; ++u) sum += exp_rel(l[j][u], by);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane_id() == 0) {
    p.sub_max[row * p.n_sub + sub] = m;
    p.sub_sum[row * p.n_sub + sub] = sum;
  }
}

// How many of s[0 .. n - 1] (n padded with zeros to a multiple of 4) are larger than x.
__device__ __forceinline__ int above(const u64* s, int n, u64 x) {
  int c = 0;
  for (int i = 0; i < n; i += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) c += s[i + u] > x;
  }
  return c;
}

constexpr int kRowThreads = 256;

// lengths of 0 count as 1
__device__ __forceinline__ double divisor(const BeamParams& a, int64_t row, int more) {
  if (!a.lengths || a.alpha == 0) return 1.0;
  const int64_t n = a.lengths[row] + more;
  return pow((double)(n > 1 ? n : 1), a.alpha);
}

template <class T>
__global__ __launch_bounds__(kRowThreads) void beam_row_kernel(BeamWork p) {
  __shared__ u64 s_best[kRowThreads], s_list[kListMost + 4];
  __shared__ int s_group[kBeamsMost];
  __shared__ double s_sum[kRowThreads / 64];
  __shared__ float s_max[kRowThreads / 64];
  __shared__ u64 s_bound;
  __shared__ int s_n;
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
      rank[0] = score / divisor(p.a, row, 0);
      sums[0] = score;
      tokens[0] = (int)p.a.end_id;
      p.count[row] = 1;
    }
    return;
  }
  // ---- lse, in an order of V alone
  float m = kNegInf;
  for (int i = t; i < p.n_sub; i += kRowThreads) m = fmaxf(m, p.sub_max[row * p.n_sub + i]);
  m = max64(max8(m));
  if (lane_id() == 0) s_max[wave_id()] = m;
  if (t == 0) s_n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 64; ++i) m = fmaxf(m, s_max[i]);
  if (!(m > kNegInf && m < kPosInf)) {  // nothing to choose (at +inf: no sum is a number)
    if (t == 0) p.count[row] = 0;
    return;
  }
  double sum = 0;
  for (int i = t; i < p.n_sub; i += kRowThreads) {
    const float mi = p.sub_max[row * p.n_sub + i];
    if (mi > kNegInf) sum += p.sub_sum[row * p.n_sub + i] * exp((double)mi - (double)m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane_id() == 0) s_sum[wave_id()] = sum;
  // ---- a bound that k groups reach: the k-th of the threads' best
  constexpr int kPer = kGroupsMost / kRowThreads;
  u64 mine[kPer], best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int g = i * kRowThreads + t;
    mine[i] = g < p.n_group ? place_of(key_of(p.group[row * p.n_group + g]), g) : 0;
    best = mine[i] > best ? mine[i] : best;
  }
  s_best[t] = best;
  if (t == 0) s_bound = 1;
  __syncthreads();
  const double rest = log(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]);  // lse - m
  if (best && above(s_best, kRowThreads, best) == k - 1) s_bound = best;
  __syncthreads();
  u64 bound = s_bound;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (mine[i] >= bound) s_list[atomicAdd(&s_n, 1)] = mine[i];
  __syncthreads();
  const int n1 = s_n;
  if (t < 4) s_list[n1 + t] = 0;
  __syncthreads();
  for (int i = t; i < n1; i += kRowThreads) {
    const u64 x = s_list[i];
    const int r = above(s_list, n1, x);
    if (r < k) s_group[r] = (int)index_at(x);
  }
  // ---- the same among the logits of the k first groups
  const int groups = n1 < k ? n1 : k, logits = groups << p.gshift;
  const T* const x = static_cast<const T*>(p.a.logits) + row * p.a.ld;
  auto place = [&](int i) -> u64 {
    const int64_t v = ((int64_t)s_group[i >> p.gshift] << p.gshift) + (i & ((1 << p.gshift) - 1));
    return v < p.a.V ? place_of(key_of((float)x[v]), v) : 0;
  };
  __syncthreads();
  best = 0;
  for (int i = t; i < logits; i += kRowThreads) {
    const u64 y = place(i);
    best = y > best ? y : best;
  }
  s_best[t] = best;
  if (t == 0) {
    s_bound = 1;
    s_n = 0;
  }
  __syncthreads();
  if (best && above(s_best, kRowThreads, best) == k - 1) s_bound = best;
  __syncthreads();
  bound = s_bound;
  for (int i = t; i < logits; i += kRowThreads) {
    const u64 y = place(i);
    if (y >= bound) {
      const int at = atomicAdd(&s_n, 1);
      if (at < kListMost) s_list[at] = y;
    }
  }
  __syncthreads();
  int n2 = s_n;
  if (n2 > kListMost) {
    // (many large logits with few threads: one round of maxima for each token)
    u64 last = ~0ull;
    n2 = 0;
    for (int r = 0; r < k; ++r) {
      best = 0;
      for (int i = t; i < logits; i += kRowThreads) {
        const u64 y = place(i);
        best = y < last && y > best ? y : best;
      }
      best = wave_max64(best);
      __syncthreads();
      if (lane_id() == 0) s_best[wave_id()] = best;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRowThreads / 64; ++i) best = s_best[i] > best ? s_best[i] : best;
      if (best == 0) break;
      if (t == 0) s_list[r] = best;
      last = best;
      n2 = r + 1;
    }
  }
  __syncthreads();
  if (t < 4) s_list[n2 + t] = 0;
  __syncthreads();
  const double by = divisor(p.a, row, 1);
  for (int i = t; i < n2; i += kRowThreads) {
    const u64 y = s_list[i];
    const int r = above(s_list, n2, y);
    if (r < k) {
      const double s = score + (((double)logit_of(key_at(y)) - (double)m) - rest);
      rank[r] = s / by;
      sums[r] = s;
      tokens[r] = (int)index_at(y);
    }
  }
  if (t == 0) p.count[row] = n2 < k ? n2 : k;
}

// One wave per sequence: a lane holds the first candidate left of its beams (lane, lane + 64, ...); k times the best of
// all goes out, and its beam's next comes up.
__global__ __launch_bounds__(64) void beam_merge_kernel(BeamWork p) {
  const int64_t b = blockIdx.x;
  const int W = p.a.W, k = p.a.k, lane = threadIdx.x;
  constexpr int kPer = kBeamsMost / 64;
  int at[kPer], n[kPer];
  double head[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int w = i * 64 + lane;
    at[i] = 0;
    n[i] = w < W ? p.count[b * W + w] : 0;
    head[i] = n[i] > 0 ? p.rank[(b * W + w) * k] : 0;
  }
  for (int r = 0; r < k; ++r) {
    // this lane's best beam (-1: none), then the wave's
    int w = -1;
    double x = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (at[i] < n[i] && (w < 0 || head[i] > x)) {
        w = i * 64 + lane;
        x = head[i];
      }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_xor(x, o);
      const int v = __shfl_xor(w, o);
      if (v >= 0 && (w < 0 || y > x || (y == x && v < w))) {
        x = y;
        w = v;
      }
    }
    const int64_t out = b * k + r;
    if (w < 0) {
      if (lane == 0) {
        p.a.token[out] = -1;
        p.a.parent[out] = -1;
        if (p.a.s64) static_cast<double*>(p.a.score)[out] = -__builtin_huge_val();
        else static_cast<float*>(p.a.score)[out] = kNegInf;
      }
      continue;
    }
    if (lane == (w & 63)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == w >> 6) {
          const int64_t from = (b * W + w) * k + at[i];
          p.a.token[out] = p.token[from];
          p.a.parent[out] = w;
          if (p.a.s64) static_cast<double*>(p.a.score)[out] = p.sum[from];
          else static_cast<float*>(p.a.score)[out] = (float)p.sum[from];
          if (++at[i] < n[i]) head[i] = p.rank[from + 1];
        }
    }
  }
}

int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

struct BeamSizes {
  int n_sub, gshift, n_group;
  int64_t sub_max, sub_sum, group, rank, sum, token, count;
  int64_t all() const { return sub_max + sub_sum + group + rank + sum + token + count; }
};
BeamSizes beam_sizes(int64_t rows, int64_t V, int k) {
  BeamSizes z;
  z.n_sub = (int)((V + kSub - 1) / kSub);
  z.gshift = V <= kSmallGroups ? 6 : 9;
  z.n_group = (int)((V + (1 << z.gshift) - 1) >> z.gshift);
  z.sub_sum = rows * z.n_sub * 8;
  z.rank = z.sum = rows * k * 8;
  z.sub_max = up8(rows * z.n_sub * 4);
  z.group = up8(rows * z.n_group * 4);
  z.token = up8(rows * k * 4);
  z.count = up8(rows * 4);
  return z;
}

template <class T>
hipError_t run(BeamWork p, hipStream_t stream) {
  const int64_t rows = p.a.B * p.a.W;
  beam_scan_kernel<T><<<(unsigned)(rows * p.n_seg), 64 * kScanWaves, 0, stream>>>(p);
  beam_row_kernel<T><<<(unsigned)rows, kRowThreads, 0, stream>>>(p);
  beam_merge_kernel<<<(unsigned)p.a.B, 64, 0, stream>>>(p);
  return hipGetLastError();
}

// ---------------------------------------------------------------- states
// A thread owns one column of V bytes of a state's beams: it reads the k parents' values before it writes any, so in
// place no other thread's reads are in the way, and a beam that keeps its parent costs nothing.
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

size_t beams_workspace_bytes(int64_t B, int W, int64_t V, int k) { return (size_t)beam_sizes(B * W, V, k).all(); }

hipError_t beams_launch(int dtype, const BeamParams& a, char* ws, hipStream_t stream) {
  if (a.B == 0) return hipSuccess;
  const int64_t rows = a.B * a.W;
  const BeamSizes z = beam_sizes(rows, a.V, a.k);
  BeamWork p{};
  p.a = a;
  p.n_sub = z.n_sub;
  p.n_seg = (z.n_sub + kScanWaves - 1) / kScanWaves;
  p.gshift = z.gshift;
  p.n_group = z.n_group;
  p.sub_sum = reinterpret_cast<double*>(ws);
  p.rank = reinterpret_cast<double*>(ws += z.sub_sum);
  p.sum = reinterpret_cast<double*>(ws += z.rank);
  p.sub_max = reinterpret_cast<float*>(ws += z.sum);
  p.group = reinterpret_cast<float*>(ws += z.sub_max);
  p.token = reinterpret_cast<int*>(ws += z.group);
  p.count = reinterpret_cast<int*>(ws += z.token);
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
