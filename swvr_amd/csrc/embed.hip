// Embedding lookup and its gradient (no counterpart in the reference, whose readout is the
// soft lookup P E of a distribution P; this is that of a token).
//
//   out[n] = scale * E[ids[n]],         gE[v] = scale * sum over n with ids[n] = v of g[n]
//
// A negative id is no token: its row of out is 0 and it adds nothing to gE.  An id of V or more reads
// nothing either; its row is NaN, so that it shows without a copy of the ids to the host.
//
// The lookup moves bytes: one 16-byte load and store per lane and step (8, 4 or one element's where rows
// are not 16-byte aligned), a row's lanes consecutive.
//
// The gradient is a sum in token order, the same on every run, without atomics on values:
//   sort_ids_kernel    the tokens in stable order of their id, and each id's segment of them (one launch);
//   embed_sum_kernel   runs of kRun sorted tokens, whatever their ids, so that an id that half the batch
//                      holds is split over many workgroups: a segment inside a run goes to its row of gE,
//                      one that crosses a run's border leaves its part in fp32; beside them, the rows
//                      without a token are written as zeros (most of gE's bytes, for a large table);
//   embed_join_kernel  adds the parts of a segment that crosses borders, in order, and writes its row.
// Up to 2048 tokens one launch does all of it, embed_direct_kernel.
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace swvr {

namespace {

template <class T> struct SumType { typedef float type; };
template <> struct SumType<double> { typedef double type; };

template <class T, int VB>
struct alignas(VB) Vec {
  static constexpr int n = VB / (int)sizeof(T);
  T v[n];
};

__device__ __forceinline__ int64_t load_id(const void* ids, int id64, int64_t i) {
  return id64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int*>(ids)[i];
}

// ---------------------------------------------------------------- lookup
// LPR lanes (a power of two up to 256) per row; a lane takes every LPR-th vector of it.
template <class T, int VB>
__global__ __launch_bounds__(256) void embed_lookup_kernel(const void* __restrict__ ids, int id64, int64_t N, int V,
                                                           const T* __restrict__ E, int64_t lde, int D, int lpr,
                                                           double scale, T* __restrict__ out, int64_t b0) {
  typedef Vec<T, VB> X;
  typedef typename SumType<T>::type A;
  const int64_t n = (b0 + blockIdx.x) * (256 / lpr) + threadIdx.x / lpr;
  if (n >= N) return;
  const int64_t id = load_id(ids, id64, n);
  const int cpr = D / X::n;
  const A s = (A)scale;
  X* dst = reinterpret_cast<X*>(out + n * D);
  if (id < 0 || id >= V) {
    X x;
#pragma unroll
    for (int i = 0; i < X::n; ++i) x.v[i] = (T)(id < 0 ? (A)0 : (A)__builtin_nanf(""));
    for (int c = threadIdx.x % lpr; c < cpr; c += lpr) dst[c] = x;
    return;
  }
  const X* src = reinterpret_cast<const X*>(E + id * lde);
  for (int c = threadIdx.x % lpr; c < cpr; c += lpr) {
    X x = src[c];
#pragma unroll
    for (int i = 0; i < X::n; ++i) x.v[i] = (T)((A)x.v[i] * s);
    dst[c] = x;
  }
}

// ---------------------------------------------------------------- sorting
// Stable order of the tokens by id in one launch: a workgroup owns consecutive ids (its rows) and scans every
// token for them, counting on the way the tokens of smaller ids, which is where its own begin; so no workgroup
// waits for another, and there is no pass per digit.  Its 16 waves take equal runs of the tokens in order.  Pass 1
// counts per (wave, row) and keeps the hits (up to kSortHits a wave); a scan over rows and waves turns the counts
// into positions; pass 2 places the hits, 64 at a time, a hit's rank among the equal ids of its 64 by ten ballots
// (one per bit of the row), so the order does not depend on any atomic's.  A wave with more hits than it kept
// scans its run again.
// The scans read every id once per workgroup, from L2, so there are few: rows for about one workgroup per CU, 256
// to 1024 (what the counts' LDS holds).  32768 tokens on 256000 ids with 256 rows each, 25 us; so, 12.
constexpr int kSortRows = 1024, kSortRowsFewest = 256, kSortWaves = 16, kSortHits = 256, kSortUnroll = 8;

template <class ID>
__global__ __launch_bounds__(64 * kSortWaves) void sort_ids_kernel(const ID* __restrict__ ids, int M, int V, int R,
                                                                   int* __restrict__ order, int* __restrict__ sid,
                                                                   int* __restrict__ seg) {
  __shared__ int cnt[kSortWaves * kSortRows];  // [wave][R]
  __shared__ int hit_i[kSortWaves][kSortHits];
  __shared__ unsigned short hit_r[kSortWaves][kSortHits];
  __shared__ int wless[kSortWaves], wtot[kSortRows / 64];
  const int t = threadIdx.x, lane = lane_id(), w = wave_id();
  const int v0 = blockIdx.x * R, rows = min(R, V - v0);
  const uint64_t below = (1ull << lane) - 1;
  int* const mine = cnt + w * R;
  for (int i = t; i < kSortWaves * R; i += 64 * kSortWaves) cnt[i] = 0;
  __syncthreads();
  const int per = (int)(((int64_t)M + 64 * kSortWaves - 1) / (64 * kSortWaves)) * 64;
  const int64_t i0 = (int64_t)w * per, i1 = i0 + per < M ? i0 + per : M;
  int less = 0, hits = 0;
  for (int64_t base = i0; base < i1; base += 64 * kSortUnroll) {
    ID x[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const int64_t i = base + u * 64 + lane;
      x[u] = i < i1 ? ids[i] : (ID)-1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      less += x[u] >= 0 && x[u] < v0;
      const bool in = x[u] >= v0 && x[u] < v0 + rows;
      const uint64_t m = __ballot(in);
      if (m == 0) continue;
      if (in) {
        const int r = (int)(x[u] - v0), at = hits + __popcll(m & below);
        atomicAdd(&mine[r], 1);
        if (at < kSortHits) {
          hit_i[w][at] = (int)(base + u * 64 + lane);
          hit_r[w][at] = (unsigned short)r;
        }
      }
      hits += __popcll(m);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) less += __shfl_xor(less, o);
  if (lane == 0) wless[w] = less;
  __syncthreads();
  int first = 0;
#pragma unroll
  for (int j = 0; j < kSortWaves; ++j) first += wless[j];
  int tot = 0, x = 0;
  if (t < R) {  // whole waves
#pragma unroll
    for (int j = 0; j < kSortWaves; ++j) tot += cnt[j * R + t];
    x = tot;  // inclusive scan over the wave's 64 rows
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (lane == 63) wtot[w] = x;
  }
  __syncthreads();
  if (t < R) {
    int s = first + x - tot;
    for (int j = 0; j < w; ++j) s += wtot[j];
    if (t < rows) seg[v0 + t] = s;
    if (t == rows - 1 && v0 + rows == V) seg[V] = s + tot;
#pragma unroll
    for (int j = 0; j < kSortWaves; ++j) {
      const int c = cnt[j * R + t];
      cnt[j * R + t] = s;
      s += c;
    }
  }
  __syncthreads();
  volatile int* const next = mine;
  auto place = [&](int i, int r, bool in) {
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 10; ++b) {
      const uint64_t m = __ballot(in && ((r >> b) & 1));
      same &= ((r >> b) & 1) ? m : ~m;
    }
    if (in) {
      const int rank = __popcll(same & below), at = next[r] + rank;
      order[at] = i;
      sid[at] = v0 + r;
      if (rank == 0) next[r] = at + __popcll(same);
    }
  };
  auto place_hits = [&](int from, int to) {
    for (int j = from; j < to; j += 64) {
      const bool in = j + lane < to;
      place(in ? hit_i[w][j + lane] : 0, in ? hit_r[w][j + lane] : 0, in);
    }
  };
  if (hits <= kSortHits) {
    place_hits(0, hits);
    return;
  }
  // The run again, its hits gathered up to whole 64s before they are placed: 262144 tokens, half of them on one
  // workgroup's ids, 324 -> 217 us (46 where they spread; a placement per 64 ids of the run, however few its hits).
  int n = 0;  // gathered, fewer than 64 between batches
  for (int64_t base = i0; base < i1; base += 64 * kSortUnroll) {
    ID x[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const int64_t i = base + u * 64 + lane;
      x[u] = i < i1 ? ids[i] : (ID)-1;
    }
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const bool in = x[u] >= v0 && x[u] < v0 + rows;
      const uint64_t m = __ballot(in);
      if (m == 0) continue;
      if (in) {
        const int at = n + __popcll(m & below);
        hit_i[w][at] = (int)(base + u * 64 + lane);
        hit_r[w][at] = (unsigned short)(x[u] - v0);
      }
      n += __popcll(m);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (n >= 64) {
        place(hit_i[w][lane], hit_r[w][lane], true);
        n -= 64;
        const int i = hit_i[w][64 + lane], r = hit_r[w][64 + lane];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        hit_i[w][lane] = i;
        hit_r[w][lane] = (unsigned short)r;
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  place_hits(0, n);
}

// ---------------------------------------------------------------- gradient
// Row of gE from an fp32 (fp64) sum.
template <class T, int VB, class A>
__device__ __forceinline__ void store_row(T* row, int c, const A (&acc)[Vec<T, VB>::n], A scale) {
  Vec<T, VB> x;
#pragma unroll
  for (int i = 0; i < Vec<T, VB>::n; ++i) x.v[i] = (T)(acc[i] * scale);
  reinterpret_cast<Vec<T, VB>*>(row)[c] = x;
}

// VB zero bytes; whole 16-byte vectors past the caches, as nothing reads them soon (V = 151936, D = 2560 in bf16: the
// launch 156 -> 152 us; rows of 8-byte vectors, D = 300 on 256000, take 31 us through the caches and 41 past them).
template <int VB>
__device__ __forceinline__ void store_zero(void* p) {
  typedef typename std::conditional<VB == 2, unsigned short, unsigned int>::type E;
  typedef E V __attribute__((ext_vector_type(VB / sizeof(E))));
  V z;
#pragma unroll
  for (int i = 0; i < (int)(VB / sizeof(E)); ++i) z[i] = 0;
  if constexpr (VB == 16)
    __builtin_nontemporal_store(z, static_cast<V*>(p));
  else
    *static_cast<V*>(p) = z;
}

struct EmbedGradKernelParams {
  const void* g;
  int64_t ldg;
  const int* order;
  const int* sid;
  const int* seg;   // [V + 1]
  int V, D, run;    // run: sorted tokens per run
  int lpr, n_ct;    // lanes per run in a workgroup, vector tiles of lpr vectors
  int n_sum;        // workgroups of the sums; the others write the rows without a token
  int dpad;         // columns of a part
  void* part;       // [runs][2][dpad]: slot 0, the segment that enters the run; slot 1, the one that leaves it
  double scale;
  void* gE;
};

// Rows without a token that one wave of the zero workgroups looks after.
constexpr int kZeroRows = 16;

template <class T, int VB>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedGradKernelParams p, int b0) {
  typedef Vec<T, VB> X;
  typedef typename SumType<T>::type A;
  const int cpr = p.D / X::n, block = b0 + (int)blockIdx.x;
  T* const gE = static_cast<T*>(p.gE);
  if (block >= p.n_sum) {
    const int v0 = ((block - p.n_sum) * 4 + wave_id()) * kZeroRows;
    const int lane = lane_id();
    // the rows' borders once, one lane each
    const int b = v0 + lane <= p.V && lane <= kZeroRows ? p.seg[v0 + lane] : 0;
    const int rows = min(kZeroRows, p.V - v0), end = __shfl_down(b, 1);  // (every lane takes part)
    const uint32_t empty = (uint32_t)__ballot(lane < rows && b == end);
    if (cpr >= 64) {
      for (int r = 0; r < rows; ++r) {
        if (!((empty >> r) & 1)) continue;
        X* row = reinterpret_cast<X*>(gE + (int64_t)(v0 + r) * p.D);
        for (int c = lane; c < cpr; c += 64) store_zero<VB>(row + c);
      }
    } else {
      X* row0 = reinterpret_cast<X*>(gE + (int64_t)v0 * p.D);
      for (int c = lane; c < rows * cpr; c += 64)
        if ((empty >> ((uint32_t)c / (uint32_t)cpr)) & 1) store_zero<VB>(row0 + c);
    }
    return;
  }
  const int rpb = 256 / p.lpr;
  const int64_t run = (int64_t)(block / p.n_ct) * rpb + threadIdx.x / p.lpr;
  const int c = (block % p.n_ct) * p.lpr + threadIdx.x % p.lpr;
  const int M = p.seg[p.V];
  const int64_t p0 = run * p.run;
  if (p0 >= M || c >= cpr) return;
  const int64_t p1 = p0 + p.run < M ? p0 + p.run : M;
  const T* const g = static_cast<const T*>(p.g);
  int cur = p.sid[p0];
  bool entered = p0 > 0 && p.sid[p0 - 1] == cur;
  const bool leaves = p1 < M && p.sid[p1] == p.sid[p1 - 1];
  A acc[X::n];
#pragma unroll
  for (int i = 0; i < X::n; ++i) acc[i] = 0;
  auto part = [&](int slot) {
    A* dst = static_cast<A*>(p.part) + (run * 2 + slot) * p.dpad + (int64_t)c * X::n;
#pragma unroll
    for (int i = 0; i < X::n; ++i) dst[i] = acc[i];
  };
  constexpr int U = 8;
  for (int64_t q = p0; q < p1; q += U) {
    X x[U];
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = q + u < p1 ? q + u : p1 - 1;
      id[u] = p.sid[at];
      x[u] = reinterpret_cast<const X*>(g + (int64_t)p.order[at] * p.ldg)[c];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q + u >= p1) break;
      if (id[u] != cur) {
        if (entered)
          part(0);
        else
          store_row<T, VB, A>(gE + (int64_t)cur * p.D, c, acc, (A)p.scale);
#pragma unroll
        for (int i = 0; i < X::n; ++i) acc[i] = 0;
        cur = id[u];
        entered = false;
      }
#pragma unroll
      for (int i = 0; i < X::n; ++i) acc[i] += (A)x[u].v[i];
    }
  }
  if (entered)
    part(0);
  else if (leaves)
    part(1);
  else
    store_row<T, VB, A>(gE + (int64_t)cur * p.D, c, acc, (A)p.scale);
}

// Parts of segments that cross runs, joined in run order.  A wave takes the run in which such a segment
// begins, 256 columns, 4 consecutive ones a lane; a workgroup's 4 waves share a segment of more than kJoinAlone parts
// (an id that fills a large share of the tokens), a quarter of its parts each.
// (32768 tokens, half of one id, D = 64: the gradient 54 -> 32 us by sharing; from 2 to 16 parts alone make no difference,
// 64 cost 24 for 19 us where such an id holds 64 parts, 4096 tokens.)
constexpr int kJoinAlone = 16, kJoinCols = 256;
template <class T>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedGradKernelParams p, int n_ct, int b0) {
  typedef typename SumType<T>::type A;
  struct alignas(16) A4 {
    A v[4];
  };
  __shared__ int s_last[4];
  __shared__ A4 s_sum[4][64];
  const int lane = lane_id(), w = wave_id(), block = b0 + (int)blockIdx.x;
  const int64_t j0 = (int64_t)(block / n_ct) * 4;
  const int d = (block % n_ct) * kJoinCols + 4 * lane;
  const int M = p.seg[p.V];
  const A* const part = static_cast<const A*>(p.part);
  // the sum of the parts of runs a .. b of the segment that begins in run j (parts are dpad wide, a multiple of 8)
  auto sum = [&](int64_t j, int64_t a, int64_t b) {
    A4 acc{{0, 0, 0, 0}};
    for (int64_t q0 = a; q0 <= b; q0 += 8) {
      A4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t q = q0 + u <= b ? q0 + u : b;
        x[u] = *reinterpret_cast<const A4*>(part + (q * 2 + (q == j)) * p.dpad + d);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (q0 + u <= b)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc.v[i] += x[u].v[i];
    }
    return acc;
  };
  auto store = [&](int v, const A4& x) {
    T* const row = static_cast<T*>(p.gE) + (int64_t)v * p.D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < p.D) row[d + i] = (T)(x.v[i] * (A)p.scale);
  };
  // the last run of the segment that begins in run j and crosses its end, or -1
  auto last_run = [&](int64_t j, int* v) -> int {
    const int64_t p0 = j * p.run, p1 = p0 + p.run;
    if (p1 >= M) return -1;
    *v = p.sid[p1 - 1];
    return p.sid[p1] == *v && p.seg[*v] >= p0 ? (p.seg[*v + 1] - 1) / p.run : -1;
  };
  int v = 0;
  const int last = last_run(j0 + w, &v);
  if (last >= 0 && last - (j0 + w) < kJoinAlone && d < p.D) store(v, sum(j0 + w, j0 + w, last));
  if (lane == 0) s_last[w] = last;
  __syncthreads();
  for (int i = 0; i < 4; ++i) {
    const int64_t j = j0 + i;
    const int b = s_last[i];
    if (b < 0 || b - j < kJoinAlone) continue;  // the same for the whole workgroup
    const int64_t n = b - j + 1, a0 = j + n * w / 4, a1 = j + n * (w + 1) / 4 - 1;
    __syncthreads();  // the sums of the segment before have been read
    if (d < p.D) s_sum[w][lane] = sum(j, a0, a1);
    __syncthreads();
    if (w == 0 && d < p.D) {
      A4 x;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x.v[c] = ((s_sum[0][lane].v[c] + s_sum[1][lane].v[c]) + s_sum[2][lane].v[c]) + s_sum[3][lane].v[c];
      store(p.sid[(j + 1) * p.run], x);
    }
  }
}

// ---------------------------------------------------------------- gradient of few tokens
// Up to kDirectMost tokens in one launch: a workgroup owns R rows of gE, sorts their tokens in LDS as sort_ids_kernel
// does (4 waves, each with a quarter of the tokens), and writes the rows, a wave each: zeros, or the sum in
// token order.  A row of more than kDirectAlone tokens is shared by the 4 waves, a quarter of its tokens each (1000 fp32
// tokens of D = 1024, ids as text has them, shared from 8, 32 and 64 on, and never: 20, 20, 24 and 31 us; 2048 with half
// of them of one id 120 for 393).
constexpr int kDirectMost = 2048, kDirectRows = 128, kDirectAlone = 32;
template <class T, int VB, class ID>
__global__ __launch_bounds__(256) void embed_direct_kernel(const ID* __restrict__ ids, int M, const T* __restrict__ g,
                                                           int64_t ldg, int V, int D, int R, double scale,
                                                           T* __restrict__ gE) {
  typedef Vec<T, VB> X;
  typedef typename SumType<T>::type A;
  constexpr int kMine = kDirectMost / 4;
  struct Sum {
    A v[X::n];
  };
  __shared__ int cnt[4][kDirectRows], seg[kDirectRows + 1], wtot[2];
  __shared__ unsigned short hit[4][kMine], order[kDirectMost];
  __shared__ unsigned char hit_r[4][kMine];
  __shared__ Sum s_sum[4][64];
  const int t = threadIdx.x, lane = lane_id(), w = wave_id();
  const int v0 = blockIdx.x * R, rows = min(R, V - v0);
  const uint64_t below = (1ull << lane) - 1;
  for (int i = t; i < 4 * kDirectRows; i += 256) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const int per = (M + 255) / 256 * 64, i0 = w * per, i1 = min(i0 + per, M);
  int hits = 0;
  for (int base = i0; base < i1; base += 256) {
    ID x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = base + u * 64 + lane < i1 ? ids[base + u * 64 + lane] : (ID)-1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = x[u] >= v0 && x[u] < v0 + rows;
      const uint64_t m = __ballot(in);
      if (m == 0) continue;
      if (in) {
        const int r = (int)(x[u] - v0), at = hits + __popcll(m & below);
        atomicAdd(&cnt[w][r], 1);
        hit[w][at] = (unsigned short)(base + u * 64 + lane);
        hit_r[w][at] = (unsigned char)r;
      }
      hits += __popcll(m);
    }
  }
  __syncthreads();
  int tot = 0, x = 0;
  if (t < kDirectRows) {
    x = tot = cnt[0][t] + cnt[1][t] + cnt[2][t] + cnt[3][t];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o);
      if (lane >= o) x += y;
    }
    if (lane == 63) wtot[w] = x;
  }
  __syncthreads();
  if (t < kDirectRows) {
    int s = x - tot + (w == 1 ? wtot[0] : 0);
    seg[t] = s;
    if (t == kDirectRows - 1) seg[kDirectRows] = s + tot;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = cnt[j][t];
      cnt[j][t] = s;
      s += c;
    }
  }
  __syncthreads();
  volatile int* const next = cnt[w];
  for (int j = 0; j < hits; j += 64) {
    const bool in = j + lane < hits;
    const int r = in ? hit_r[w][j + lane] : 0;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 7; ++b) {
      const uint64_t m = __ballot(in && ((r >> b) & 1));
      same &= ((r >> b) & 1) ? m : ~m;
    }
    if (in) {
      const int rank = __popcll(same & below), at = next[r] + rank;
      order[at] = hit[w][j + lane];
      if (rank == 0) next[r] = at + __popcll(same);
    }
  }
  __syncthreads();
  const int cpr = D / X::n;
  // the sum of the tokens a .. b - 1 of the order in vector c
  auto sum = [&](int a, int b, int c) {
    Sum acc;
#pragma unroll
    for (int i = 0; i < X::n; ++i) acc.v[i] = 0;
    for (int q = a; q < b; q += 8) {
      X y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        y[u] = reinterpret_cast<const X*>(g + (int64_t)order[q + u < b ? q + u : b - 1] * ldg)[c];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (q + u < b)
#pragma unroll
          for (int i = 0; i < X::n; ++i) acc.v[i] += (A)y[u].v[i];
    }
    return acc;
  };
  bool shared_rows = false;
  for (int r = w; r < rows; r += 4) {
    const int a = seg[r], b = seg[r + 1];
    if (b - a > kDirectAlone) {
      shared_rows = true;
      continue;
    }
    T* const row = gE + (int64_t)(v0 + r) * D;
    if (a == b) {
      for (int c = lane; c < cpr; c += 64) store_zero<VB>(row + (int64_t)c * X::n);
      continue;
    }
    for (int c = lane; c < cpr; c += 64) {
      const Sum acc = sum(a, b, c);
      store_row<T, VB, A>(row, c, acc.v, (A)scale);
    }
  }
  if (!__syncthreads_or(shared_rows)) return;
  for (int r = 0; r < rows; ++r) {
    const int a = seg[r], n = seg[r + 1] - a;
    if (n <= kDirectAlone) continue;  // the same for the whole workgroup
    T* const row = gE + (int64_t)(v0 + r) * D;
    for (int c0 = 0; c0 < cpr; c0 += 64) {
      const int c = c0 + lane;
      if (c < cpr) s_sum[w][lane] = sum(a + n * w / 4, a + n * (w + 1) / 4, c);
      __syncthreads();
      if (w == 0 && c < cpr) {
        Sum acc = s_sum[0][lane];
#pragma unroll
        for (int j = 1; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < X::n; ++i) acc.v[i] += s_sum[j][lane].v[i];
        store_row<T, VB, A>(row, c, acc.v, (A)scale);
      }
      __syncthreads();
    }
  }
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int elem_bytes(int dtype) { return dtype == kF64 ? 8 : dtype == kF32 ? 4 : 2; }

// Largest vector (16, 8, 4, ... bytes) that divides every row and base.
int vec_bytes(int eb, int64_t D, int64_t ld, const void* a, const void* b) {
  int vb = 16;
  const uintptr_t x = (uintptr_t)(D * eb) | (uintptr_t)(ld * eb) | (uintptr_t)a | (uintptr_t)b;
  while (vb > eb && (x & (vb - 1))) vb /= 2;
  return vb;
}

// Lanes per row: the most (up to 256, a wave at least for rows of 64 vectors) that leave under a tenth idle,
// or the fewest idle.
int lanes_per_row(int cpr) {
  int best = 8, waste = 1 << 30;
  for (int l = 256; l >= 8; l /= 2) {
    const int idle = (cpr + l - 1) / l * l - cpr;
    if (idle * 10 <= cpr) return l;
    if (idle < waste) {
      waste = idle;
      best = l;
    }
  }
  return best;
}

// f(element type, vector bytes) for a dtype tag and vector width.
template <class F>
hipError_t dispatch(int dtype, int vb, F&& f) {
  auto by_vb = [&](auto t) -> hipError_t {
    typedef decltype(t) T;
    if (vb == 16) return f(t, std::integral_constant<int, 16>());
    if (vb == 8) return f(t, std::integral_constant<int, 8>());
    if constexpr (sizeof(T) <= 4)
      if (vb == 4) return f(t, std::integral_constant<int, 4>());
    if constexpr (sizeof(T) == 2)
      if (vb == 2) return f(t, std::integral_constant<int, 2>());
    return hipErrorInvalidValue;
  };
  switch (dtype) {
    case kBF16: return by_vb((bf16_t)0.f);
    case kF16: return by_vb((f16_t)0.f);
    case kF32: return by_vb(0.f);
    case kF64: return by_vb(0.0);
    default: return hipErrorInvalidValue;
  }
}

// Sorted tokens per run: 64, and 32 and 16 for the fewer tokens that would not fill the chip so.  A lane walks a run's
// rows in turn, 8 in flight, and a longer run leaves fewer parts to join.  The sums and the join in bf16 on 50000 rows,
// with 16, 32 and 64: 4096 tokens, D = 64 17, 17 and 23 us, D = 1024 26, 28 and 35; 16384, D = 300 20, 21 and 28;
// 65536, D = 300 33, 32 and 33, D = 1024 53, 49 and 46.  (So 32 would still serve 16384 to 32768 tokens better.)
int run_of(int64_t M) { return M >= 16384 ? 64 : M >= 4096 ? 32 : 16; }

}  // namespace

hipError_t embed_lookup_launch(const EmbedParams& p, hipStream_t stream) {
  if (p.N == 0 || p.D == 0) return hipSuccess;
  const int eb = elem_bytes(p.dtype), vb = vec_bytes(eb, p.D, p.lde, p.E, p.out);
  return dispatch(p.dtype, vb, [&](auto t, auto w) -> hipError_t {
    typedef decltype(t) T;
    constexpr int VB = decltype(w)::value;
    const int lpr = lanes_per_row(p.D / (VB / (int)sizeof(T))), rpb = 256 / lpr;
    timing_begin(kKindEmbed, stream);
    const hipError_t e = launch_in_parts((p.N + rpb - 1) / rpb, 256, [&](int64_t b0, unsigned n) {
      embed_lookup_kernel<T, VB><<<n, 256, 0, stream>>>(p.ids, p.id64, p.N, p.V, static_cast<const T*>(p.E), p.lde, p.D,
                                                        lpr, p.scale, static_cast<T*>(p.out), b0);
    });
    timing_end(kKindEmbed, stream);
    return e;
  });
}

hipError_t sort_ids(const void* ids, int id64, int M, int V, int* order, int* sid, int* seg, hipStream_t stream) {
  if (V == 0) return hipSuccess;
  int R = kSortRowsFewest;
  while (R < kSortRows && (int64_t)R * 256 < V) R *= 2;
  const unsigned blocks = (unsigned)(((int64_t)V + R - 1) / R);
  timing_begin(kKindSortIds, stream);
  if (id64)
    sort_ids_kernel<int64_t><<<blocks, 64 * kSortWaves, 0, stream>>>(static_cast<const int64_t*>(ids), M, V, R,
                                                                      order, sid, seg);
  else
    sort_ids_kernel<int><<<blocks, 64 * kSortWaves, 0, stream>>>(static_cast<const int*>(ids), M, V, R, order, sid,
                                                                 seg);
  timing_end(kKindSortIds, stream);
  return hipGetLastError();
}

namespace {
// order [N], sid [N], seg [V + 1] in one buffer
struct Sorted {
  int *order, *sid, *seg;
};
Sorted sorted_in(int* p, int64_t N) { return {p, p + N, p + 2 * N}; }

template <class T, int VB>
hipError_t launch_direct(const EmbedParams& p, hipStream_t stream) {
  // rows for about 1024 workgroups, up to what a workgroup's LDS holds
  int R = 4;
  while (R < kDirectRows && (int64_t)R * 1024 < p.V) R *= 2;
  const unsigned blocks = (unsigned)(((int64_t)p.V + R - 1) / R);
  const T* const g = static_cast<const T*>(p.g);
  T* const gE = static_cast<T*>(p.gE);
  timing_begin(kKindEmbed, stream);
  if (p.id64)
    embed_direct_kernel<T, VB, int64_t><<<blocks, 256, 0, stream>>>(static_cast<const int64_t*>(p.ids), (int)p.N, g,
                                                                     p.ldg, p.V, p.D, R, p.scale, gE);
  else
    embed_direct_kernel<T, VB, int><<<blocks, 256, 0, stream>>>(static_cast<const int*>(p.ids), (int)p.N, g, p.ldg,
                                                                 p.V, p.D, R, p.scale, gE);
  timing_end(kKindEmbed, stream);
  return hipGetLastError();
}
}  // namespace

size_t embed_sorted_ints(int64_t N, int64_t V) { return N <= kDirectMost ? 0 : (size_t)(2 * N + V + 1); }

hipError_t embed_sort(const EmbedParams& p, int* sorted, hipStream_t stream) {
  if (p.N <= kDirectMost) return hipSuccess;
  const Sorted z = sorted_in(sorted, p.N);
  return sort_ids(p.ids, p.id64, (int)p.N, p.V, z.order, z.sid, z.seg, stream);
}

size_t embed_grad_workspace_bytes(int dtype, int64_t N, int64_t V, int64_t D) {
  if (N <= kDirectMost) return 0;
  const int64_t run = run_of(N), runs = (N + run - 1) / run, dpad = (D + 7) / 8 * 8;
  return align256(embed_sorted_ints(N, V) * 4) + align256((size_t)runs * 2 * dpad * (dtype == kF64 ? 8 : 4));
}

hipError_t embed_grad_launch(const EmbedParams& p, const int* sorted, char* ws, hipStream_t stream) {
  if (p.V == 0 || p.D == 0) return hipSuccess;
  const int eb = elem_bytes(p.dtype), vb = vec_bytes(eb, p.D, p.ldg, p.g, p.gE);
  hipError_t e;
  if (p.N <= kDirectMost)
    return dispatch(p.dtype, vb, [&](auto t, auto w) { return launch_direct<decltype(t), decltype(w)::value>(p, stream); });
  // the workspace: the parts, then the sorted order of a caller that has none
  const int64_t run = run_of(p.N), runs = (p.N + run - 1) / run;
  const int dpad = (p.D + 7) / 8 * 8;
  if (!sorted) {
    int* const own = reinterpret_cast<int*>(ws + align256((size_t)runs * 2 * dpad * (p.dtype == kF64 ? 8 : 4)));
    if ((e = embed_sort(p, own, stream)) != hipSuccess) return e;
    sorted = own;
  }
  const Sorted z = sorted_in(const_cast<int*>(sorted), p.N);
  EmbedGradKernelParams k{};
  k.g = p.g;
  k.ldg = p.ldg;
  k.order = z.order;
  k.sid = z.sid;
  k.seg = z.seg;
  k.V = p.V;
  k.D = p.D;
  k.run = (int)run;
  k.dpad = dpad;
  k.part = ws;
  k.scale = p.scale;
  k.gE = p.gE;
  e = dispatch(p.dtype, vb, [&](auto t, auto w) -> hipError_t {
    typedef decltype(t) T;
    constexpr int VB = decltype(w)::value;
    const int cpr = p.D / (VB / (int)sizeof(T));
    const int l = lanes_per_row(cpr);
    k.lpr = l;
    k.n_ct = (cpr + l - 1) / l;
    const int64_t sums = (runs + 256 / l - 1) / (256 / l) * k.n_ct;
    const int64_t zeros = ((int64_t)p.V + 4 * kZeroRows - 1) / (4 * kZeroRows);
    if (sums + zeros > INT32_MAX) return hipErrorInvalidValue;
    k.n_sum = (int)sums;
    timing_begin(kKindEmbed, stream);
    const hipError_t launched = launch_in_parts(sums + zeros, 256, [&](int64_t b0, unsigned n) {
      embed_sum_kernel<T, VB><<<n, 256, 0, stream>>>(k, (int)b0);
    });
    timing_end(kKindEmbed, stream);
    return launched;
  });
  if (e != hipSuccess || runs < 2) return e;
  const int n_ct = (p.D + kJoinCols - 1) / kJoinCols;
  const int64_t blocks = (runs + 3) / 4 * n_ct;
  if (blocks > INT32_MAX) return hipErrorInvalidValue;
  timing_begin(kKindEmbed, stream);
  e = launch_in_parts(blocks, 256, [&](int64_t b0, unsigned n) {
    switch (p.dtype) {
      case kBF16: embed_join_kernel<bf16_t><<<n, 256, 0, stream>>>(k, n_ct, (int)b0); break;
      case kF16: embed_join_kernel<f16_t><<<n, 256, 0, stream>>>(k, n_ct, (int)b0); break;
      case kF32: embed_join_kernel<float><<<n, 256, 0, stream>>>(k, n_ct, (int)b0); break;
      default: embed_join_kernel<double><<<n, 256, 0, stream>>>(k, n_ct, (int)b0); break;
    }
  });
  timing_end(kKindEmbed, stream);
  return e;
}

}  // namespace swvr
