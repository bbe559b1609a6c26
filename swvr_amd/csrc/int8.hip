// The head in 8-bit integers (no counterpart in the reference): rows quantised with a scale each, and logits
//
//   out[n, v] = logit_scale sh[n] sw[v] sum_k qh[n, k] qw[v, k] + bias[v],
//
// the sum in 32-bit integers, exact for K up to 2^17 (127 127 2^17 < 2^31), so the result does not depend on how the
// reduction is split.
//
// Rows are kept in the order in which the matrix cores take them (launch.hpp, kInt8Block): an operand of
// v_mfma_i32_32x32x32_i8 is 16 consecutive bytes per lane, lane l's row l % 32 and values 16 (l / 32) on, which is
// 1 KB in one piece for the wave, from memory as from LDS, free of bank conflicts without a swizzle.
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace swvr {

// Loads of R rows (whole 32-row groups) of an image, a slice of 64 values at a time.
template <int R, int NT>
struct I8Tile {
  typedef I8Tile Layout;
  static constexpr int BYTES = R * 64, NI = BYTES / (NT * 16), NI_MIN = NI;
  static_assert(R % 32 == 0 && BYTES % (NT * 16) == 0, "whole groups, whole workgroup loads");
  const char* base;
  uint32_t off[NI];
  __device__ __forceinline__ void setup(const char* image, int row0, int S) {
    base = image + (int64_t)(row0 >> 5) * S * kInt8Block;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int lin = i * NT + (int)threadIdx.x;  // 16-byte chunk of the tile
      off[i] = (uint32_t)((lin / 128) * S * (int)kInt8Block + (lin % 128) * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t lds, int s) const {
    dma_n<NI, NT * 16>(make_rsrc(base + (int64_t)s * kInt8Block), off, lds + wave_id() * 1024);
  }
};
template <int R, int NT, int F, int J>
struct OpOffsets<I8Tile<R, NT>, F, J> {
  uint32_t off;
  __device__ __forceinline__ void init(int row0) { off = (row0 >> 5) * (int)kInt8Block + lane_id() * 16; }
  __device__ __forceinline__ i32x4_t read(const char* stage, int j, int f) const {
    return *reinterpret_cast<const i32x4_t*>(stage + off + f * (int)kInt8Block + j * 1024);
  }
};

namespace {

// ---------------------------------------------------------------- quantisation
constexpr float kTinyAmax = 1e-30f;

// 16 consecutive values of a row from k on, 0 past K, as they are stored: loads of several go out before the first is
// used.  Rows begin at any element (K odd).
template <class Src>
struct Sixteen {
  typedef Src V __attribute__((ext_vector_type(8)));
  V v[2];
  __device__ __forceinline__ void load(const Src* row, int k, int K) {
    typedef V __attribute__((aligned(sizeof(Src)))) Unaligned;
    if (k + 16 <= K) {
#pragma unroll
      for (int h = 0; h < 2; ++h) v[h] = *reinterpret_cast<const Unaligned*>(row + k + 8 * h);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = k + i < K ? row[k + i] : (Src)0.f;
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i / 8][i % 8]; }
};

// The largest magnitude of a row by its bits, so that an infinity or a NaN is larger than any number; 2-byte types two
// at a time.
template <class Src>
struct Magnitude {
  typedef uint16_t U2 __attribute__((ext_vector_type(2)));
  uint32_t m = 0;
  __device__ __forceinline__ void add(const Sixteen<Src>& y) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2 * (int)sizeof(Src); ++i) {
        uint32_t w;
        __builtin_memcpy(&w, reinterpret_cast<const char*>(&y.v[h]) + 4 * i, 4);
        if constexpr (sizeof(Src) == 2) {
          m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(U2, m), __builtin_bit_cast(U2, w & 0x7fff7fffu)));
        } else {
          const uint32_t b = w & 0x7fffffffu;
          m = b > m ? b : m;
        }
      }
  }
  // as the bits of an fp32
  __device__ __forceinline__ uint32_t bits() const {
    if constexpr (sizeof(Src) == 4) {
      return m;
    } else {
      const uint16_t a = (uint16_t)m, b = (uint16_t)(m >> 16);
      return __float_as_uint((float)__builtin_bit_cast(Src, a > b ? a : b)) & 0x7fffffffu;
    }
  }
};

// x / s to the nearest whole number, halves to even, as the exact quotient has it: the product with 1 / s may fall
// on the other side of a border, which the remainder x - q s shows (exact in one fma: where it is near s / 2 it is a
// multiple of half a unit of s's last place, and below 2^24 of them).
__device__ __forceinline__ int quantize(float x, float s, float inv, float half) {
  const float q = rintf(x * inv);
  const float d = fmaf(-q, s, x);
  const int n = (int)q, up = d > 0.f ? 1 : -1;
  const float a = fabsf(d);
  return a > half || (a == half && (n & 1)) ? n + up : n;
}
// 16 of them as bytes.  The sum with 1.5 2^23 is rounded to a whole number, whose low byte is the value; only a lane
// with a remainder of half a step or more needs a second look.
template <class Src>
__device__ __forceinline__ uint4 quantize16(const Sixteen<Src>& x, float s, float inv, float half) {
  constexpr float kRound = 12582912.f;
  uint32_t w[4];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float y = fmaf(x[4 * i + u], inv, kRound);
      far = fmaxf(far, fabsf(fmaf(kRound - y, s, x[4 * i + u])));
      b[u] = __float_as_uint(y);
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400);
    w[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100);
  }
  if (far >= half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) w[i] |= (uint32_t)(quantize(x[4 * i + u], s, inv, half) & 255) << (8 * u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// TPR threads a row, a wave for many rows and a workgroup for few, each with NC pieces of 16 values in registers, so
// that rows of up to 16 NC TPR values are read once (longer ones twice).  A piece goes out as one 16-byte chunk of the
// image; the workgroup's rows are neighbours in it, 8 of them 128 bytes in a row.  Bound by reading x and writing a byte
// a value: 151936 x 2560 in bf16 221 us, 5.3 TB/s, again and again; 240 after a dequantisation, whose stores fill the
// caches.  (8 threads a row, whose chunks go out together without LDS but who read their rows twice: 415 us.)
constexpr int kManyRows = 8;
template <class Src, int TPR, int NC>
__global__ __launch_bounds__(TPR == 64 ? 64 * kManyRows : TPR) void int8_quantize_kernel(
    const Src* __restrict__ x, int64_t ld, int64_t R, int K, int S, char* __restrict__ image, float* __restrict__ scale) {
  __shared__ uint32_t s_max[4];
  const int64_t r = TPR == 64 ? (int64_t)xcd_swizzle(blockIdx.x, gridDim.x) * kManyRows + wave_id() : (int64_t)blockIdx.x;
  const int j = TPR == 64 ? lane_id() : (int)threadIdx.x;
  const Src* row = x + r * ld;
  Sixteen<Src> v[NC];
  Magnitude<Src> most;
  if (r < R) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = (c * TPR + j) * 16;
      if (c * TPR * 16 < K) v[c].load(row, k < K ? k : K, K);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c * TPR * 16 < K) most.add(v[c]);
    for (int k = (NC * TPR + j) * 16; k < K; k += TPR * 16) {
      Sixteen<Src> y;
      y.load(row, k, K);
      most.add(y);
    }
  }
  uint32_t m = most.bits();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_xor(m, o);
    m = y > m ? y : m;
  }
  if constexpr (TPR == 256) {
    if (lane_id() == 0) s_max[wave_id()] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) m = s_max[i] > m ? s_max[i] : m;
  }
  const bool fine = m < 0x7f800000u;
  const float s = fmaxf(__uint_as_float(m), kTinyAmax) * (1.f / 127.f), inv = 1.f / s, half = 0.5f * s;
  if (j == 0 && r < R) scale[r] = fine ? s : __uint_as_float(0x7fc00000u);
  const bool any = r < R && fine;
  char* out = image + (r >> 5) * S * kInt8Block + (r & 31) * 16;
  auto chunk = [&](const Sixteen<Src>& y, int k) {
    return any && k < K ? quantize16(y, s, inv, half) : make_uint4(0, 0, 0, 0);
  };
  if constexpr (TPR == 64) {
    // the 8 rows' chunks of 16 values meet in LDS (row w's of chunk c in place w ^ c % 8 of 8: no bank conflicts), and
    // 8 lanes write their 128 bytes
    __shared__ uint4 s_out[NC * 64 * kManyRows];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = c * 64 + j;
      if (i * 16 < S * 64) s_out[i * kManyRows + (wave_id() ^ (i % kManyRows))] = chunk(v[c], i * 16);
    }
    __syncthreads();
    char* const to = image + (r >> 5) * S * kInt8Block + (r - wave_id() & 31) * 16;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int q = c * 64 * kManyRows + (int)threadIdx.x, i = q / kManyRows, w = q % kManyRows;
      if (i * 16 < S * 64) *reinterpret_cast<uint4*>(to + (int64_t)i * 512 + w * 16) = s_out[i * kManyRows + (w ^ (i % kManyRows))];
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int k = (c * TPR + j) * 16;
      if (k < S * 64) *reinterpret_cast<uint4*>(out + (int64_t)(k >> 4) * 512) = chunk(v[c], k);
    }
  }
  for (int k = (NC * TPR + j) * 16; k < S * 64; k += TPR * 16) {
    Sixteen<Src> y;
    if (any) y.load(row, k < K ? k : K, K);
    *reinterpret_cast<uint4*>(out + (int64_t)(k >> 4) * 512) = chunk(y, k);
  }
}

// Rows of integers [R][ld] into an image, 8 threads a row: 151936 x 2560 in 140 to 155 us, 5.6 to 5.0 TB/s of what is read and
// written.
__global__ __launch_bounds__(256) void int8_pack_kernel(const int8_t* __restrict__ q, int64_t ld, int64_t R, int K, int S,
                                                        int vec, char* __restrict__ image) {
  const int64_t r = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  const int8_t* row = q + r * ld;
  char* out = image + (r >> 5) * S * kInt8Block + (r & 31) * 16;
  for (int k = (threadIdx.x % 8) * 16; k < S * 64; k += 128) {
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < R && vec && k + 16 <= K) {
      w = *reinterpret_cast<const uint4*>(row + k);
    } else if (r < R) {
      int8_t b[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) b[i] = k + i < K ? row[k + i] : (int8_t)0;
      __builtin_memcpy(&w, b, 16);
    }
    *reinterpret_cast<uint4*>(out + (int64_t)(k >> 4) * 512) = w;
  }
}

// The values that an image stands for, in fp32 [R][K]: 32 rows x kUnpackK values through LDS, so that the image comes
// in and rows go out in long pieces (16 bytes a lane; a chunk's 512 bytes padded to 528: no bank conflicts).  151936 x
// 2560 in 334 to 344 us, 5.8 to 5.7 TB/s.
constexpr int kUnpackK = 256;
__global__ __launch_bounds__(256) void int8_unpack_kernel(const char* __restrict__ image, const float* __restrict__ scale,
                                                          int64_t R, int K, int S, int pieces, float* __restrict__ out) {
  constexpr int kPitch = 528;
  __shared__ __attribute__((aligned(16))) char s_q[kUnpackK / 16 * kPitch];
  const int64_t r0 = blockIdx.x / pieces * 32;
  const int k0 = blockIdx.x % pieces * kUnpackK;
  const char* in = image + (r0 >> 5) * S * kInt8Block + (int64_t)(k0 >> 4) * 512;
#pragma unroll
  for (int i = 0; i < kUnpackK / 16 * 32 / 256; ++i) {
    const int c = i * 256 + threadIdx.x;  // chunk c / 32 of row c % 32
    if (k0 + (c / 32) * 16 < S * 64)
      *reinterpret_cast<uint4*>(s_q + (c / 32) * kPitch + (c % 32) * 16) = *reinterpret_cast<const uint4*>(in + c * 16);
  }
  __syncthreads();
  const int k = k0 + lane_id() * 4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = wave_id() * 8 + i;
    if (r0 + row >= R || k >= K) continue;
    const int w = *reinterpret_cast<const int*>(s_q + (lane_id() / 4) * kPitch + row * 16 + (lane_id() % 4) * 4);
    const float s = scale[r0 + row];
    typedef float F4 __attribute__((ext_vector_type(4)));
    typedef F4 __attribute__((aligned(4))) Unaligned;
    F4 y;
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = (float)(w << (24 - 8 * u) >> 24) * s;
    float* to = out + (r0 + row) * K + k;
    if (k + 4 <= K) {
      *reinterpret_cast<Unaligned*>(to) = y;
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < K) to[u] = y[u];
    }
  }
}

// ---------------------------------------------------------------- logits
__device__ __forceinline__ float bias_at(const Int8Params& p, int v) {
  if (!p.bias || v >= p.V) return 0.f;
  if (p.b_dtype == kF32) return static_cast<const float*>(p.bias)[v];
  if (p.b_dtype == kF16) return (float)static_cast<const f16_t*>(p.bias)[v];
  return (float)static_cast<const bf16_t*>(p.bias)[v];
}
__device__ __forceinline__ float wscale_at(const Int8Params& p, int v) { return v < p.V ? p.w_scale[v] : 0.f; }

// logit_scale sh sw sum + bias.  The scales' product may leave fp32 where the logit does not (2^-106 sh of a token of zeros
// times sw of a row of zeros; rows of 1e36 times a scale of 1e4, with a sum of 0): then in fp64, which holds all but the last
// bits of it.  Whether that is so depends on the two scales alone.
__device__ __forceinline__ bool holds(float x) {
  x = fabsf(x);
  return x >= 0x1p-126f && x < kPosInf;
}
__device__ __forceinline__ float near_logit(int sum, float csh, float sw, float bias) { return fmaf((float)sum, csh * sw, bias); }
__device__ __forceinline__ float far_logit(int sum, float c, float sh, float sw, float bias) {
  const float csh = c * sh;
  if (holds(csh) && holds(csh * sw)) [[likely]]
    return near_logit(sum, csh, sw, bias);
  return (float)fma((double)c * (double)sh * (double)sw, (double)sum, (double)bias);
}

// Up to 32 NB tokens on few rows: a workgroup takes 32 G of W's rows, its four waves a quarter of the reduction each,
// operands straight from memory; the quarters are added in LDS.  Bound by a round trip or two to memory: K = 4096, V =
// 16000, one token 11.1 us with the quantisation.
template <class Out, int NB, int G, int U>
__global__ __launch_bounds__(256) void int8_few_kernel(Int8Params p) {
  constexpr int kRegs = G * NB * 16, kPitch = 65;
  __shared__ int s_part[4][kRegs * kPitch];
  const int lane = lane_id(), w = wave_id();
  const int v0 = blockIdx.x * 32 * G;
  i32x16_t acc[G][NB];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[g][b][r] = 0;
  const int s0 = w * p.S / 4, s1 = (w + 1) * p.S / 4;
  const int64_t rows = (int64_t)p.S * kInt8Block;  // bytes of 32 rows
  const char* const wp = p.w + (int64_t)(v0 >> 5) * rows + lane * 16;
  const char* const hp = p.h + lane * 16;
  auto load = [&](const char* q, int g, int s, int j) {
    return *reinterpret_cast<const i32x4_t*>(q + g * rows + (int64_t)s * kInt8Block + j * 1024);
  };
  int s = s0;
  for (; s + U <= s1; s += U) {
    i32x4_t a[U][G][2], h[U][NB][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int g = 0; g < G; ++g) a[u][g][j] = load(wp, g, s + u, j);
#pragma unroll
        for (int b = 0; b < NB; ++b) h[u][b][j] = load(hp, b, s + u, j);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int b = 0; b < NB; ++b) mfma_k16(acc[g][b], a[u][g][j], h[u][b][j]);
  }
  for (; s < s1; ++s)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int b = 0; b < NB; ++b) mfma_k16(acc[g][b], load(wp, g, s, j), load(hp, b, s, j));
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) s_part[w][((g * NB + b) * 16 + r) * kPitch + lane] = acc[g][b][r];
  __syncthreads();
  Out* const out = static_cast<Out*>(p.out);
  // a thread per vocabulary row of a token: row i of a group is in register i / 8 * 4 + i % 4 of lanes 32 (i / 4 % 2) on
  const int i = threadIdx.x % (32 * G), g = i / 32, row = i % 32;
  const int v = v0 + i;
  const float sw = wscale_at(p, v), bias = bias_at(p, v);
  for (int n = threadIdx.x / (32 * G); n < p.N; n += 256 / (32 * G)) {
    const int at = ((g * NB + n / 32) * 16 + row / 8 * 4 + row % 4) * kPitch + (row / 4 % 2) * 32 + n % 32;
    const int sum = s_part[0][at] + s_part[1][at] + s_part[2][at] + s_part[3][at];
    if (v < p.V) out[(int64_t)n * p.V + v] = (Out)far_logit(sum, p.scale, p.h_scale[n], sw, bias);
  }
}

// 16 bytes of logits at any element.
template <class Out>
struct __attribute__((packed, aligned(sizeof(Out)))) OutChunk {
  Out v[16 / sizeof(Out)];
};

// A wave's 32 FM vocabulary rows (from v0) x 32 FN tokens (from n0), through `room` (ROOM bytes of LDS, this wave's): a
// lane holds 4 rows of a token, and goes out with 16 bytes of a token's 256 (128 with fewer rows or less room).
template <class Out, int FM, int FN, int ROOM, bool FAR>
__device__ __forceinline__ void store_tile(const Int8Params& p, const i32x16_t (&acc)[FM][FN], char* room,
                                           const float* scale, const float* bias, int v0, int n0) {
  constexpr int E = (int)sizeof(Out), kFit = ROOM >= 32 * (256 + 16) ? 8 / E : 4 / E;
  constexpr int FP = FM < kFit ? FM : kFit;  // blocks of 32 rows in a piece
  constexpr int kBytes = FP * 32 * E, kPitch = kBytes + 16, kLanes = kBytes / 16;
  static_assert(FM % FP == 0 && 32 * kPitch <= ROOM, "whole pieces, which fit");
  struct alignas(4 * E) Four {
    Out v[4];
  };
  const int lane = lane_id();
#pragma unroll
  for (int fn = 0; fn < FN; ++fn) {
    const int nb = n0 + fn * 32, n = nb + (lane & 31);
    const float sh = n < p.N ? p.h_scale[n] : 0.f, csh = p.scale * sh;
#pragma unroll
    for (int f0 = 0; f0 < FM; f0 += FP) {
#pragma unroll
      for (int f = 0; f < FP; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int c = f * 32 + 8 * g + (lane >> 5) * 4;
          const float4 sw = *reinterpret_cast<const float4*>(scale + f0 * 32 + c);
          const float4 b = *reinterpret_cast<const float4*>(bias + f0 * 32 + c);
          const float sws[4] = {sw.x, sw.y, sw.z, sw.w}, bs[4] = {b.x, b.y, b.z, b.w};
          Four y;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int sum = acc[f0 + f][fn][4 * g + i];
            y.v[i] = (Out)(FAR ? far_logit(sum, p.scale, sh, sws[i], bs[i]) : near_logit(sum, csh, sws[i], bs[i]));
          }
          *reinterpret_cast<Four*>(room + (lane & 31) * kPitch + c * E) = y;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < kLanes / 2; ++i) {
        const int t = i * (64 / kLanes) + lane / kLanes, at = (lane % kLanes) * 16;
        const int v = v0 + f0 * 32 + at / E;
        const OutChunk<Out> y = *reinterpret_cast<const OutChunk<Out>*>(__builtin_assume_aligned(room + t * kPitch + at, 16));
        if (nb + t >= p.N) continue;
        Out* const to = static_cast<Out*>(p.out) + (int64_t)(nb + t) * p.V + v;
        if (v + 16 / E <= p.V) {
          if (p.lines)
            __builtin_nontemporal_store(__builtin_bit_cast(i32x4_t, y), reinterpret_cast<i32x4_t*>(to));
          else
            *reinterpret_cast<OutChunk<Out>*>(to) = y;
        } else {
#pragma unroll
          for (int u = 0; u < 16 / E; ++u)
            if (v + u < p.V) to[u] = y.v[u];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// Whether a product of a wave's scales may leave fp32, which is where its logits take the long way.  None does with |sw| in
// 2^-107 (what a row of zeros has) .. 2^60 and |c sh| in 2^-19 .. 2^60, or with 2^-16 .. and 2^-110 .. (a token of zeros).
template <int FM, int FN>
struct Scales {
  float w[(FM + 1) / 2], h[(FN + 1) / 2];
  __device__ __forceinline__ void load(const Int8Params& p, int v0, int n0) {
#pragma unroll
    for (int i = 0; i < (FM + 1) / 2; ++i) w[i] = p.w_scale[min(v0 + (i * 64 + lane_id()) % (32 * FM), p.V - 1)];
#pragma unroll
    for (int i = 0; i < (FN + 1) / 2; ++i) h[i] = p.h_scale[min(n0 + (i * 64 + lane_id()) % (32 * FN), p.N - 1)];
  }
  __device__ __forceinline__ bool far(float c) const {
    bool small = false, any = false;
#pragma unroll
    for (int i = 0; i < (FM + 1) / 2; ++i) {
      small |= fabsf(w[i]) < 0x1p-16f;
      any |= !(fabsf(w[i]) >= 0x1p-107f && fabsf(w[i]) <= 0x1p60f);
    }
    const float least = __any(small) ? 0x1p-19f : 0x1p-110f;
#pragma unroll
    for (int i = 0; i < (FN + 1) / 2; ++i) any |= !(fabsf(c * h[i]) >= least && fabsf(c * h[i]) <= 0x1p60f);
    return __any(any);
  }
};

// Many tokens: BV x BM tiles of WV x WT waves, the readout's reduction loop (tile_reduce) on integer operands.  Up to some
// 300 tokens bound by reading W (48 tokens, K = 4096, V = 128256: 101 us, 5.2 TB/s), beyond by the power that matrix cores
// take: 8192 tokens 3430 to 3660 us, 2510 to 2350 TOP/s, at 1.4 to 1.5 GHz with the matrix cores busy in 74% of the
// cycles; the loop alone would take 3130.
template <class Out, int BV, int BM, int WV, int WT, int NS>
__global__ __launch_bounds__(64 * WV * WT) void int8_tile_kernel(Int8Params p) {
  constexpr int NT = 64 * WV * WT, FM = BV / WV / 32, FN = BM / WT / 32;
  typedef I8Tile<BV, NT> TA;
  typedef I8Tile<BM, NT> TB;
  constexpr int SB = TA::BYTES + TB::BYTES, L = TA::NI + TB::NI;
  __shared__ __attribute__((aligned(1024))) char smem[NS * SB];
  __shared__ __attribute__((aligned(16))) float s_scale[BV], s_bias[BV];
  const int w = wave_id(), wv = w / WT, wt = w % WT;
  int vt, tb;
  grouped_tile(blockIdx.x, p.n_vt, p.n_tb, &vt, &tb);
  const int v0 = vt * BV + wv * (BV / WV), n0 = tb * BM + wt * (BM / WT);  // the wave's
  for (int i = threadIdx.x; i < BV; i += NT) {
    s_scale[i] = wscale_at(p, vt * BV + i);
    s_bias[i] = bias_at(p, vt * BV + i);
  }
  // Scales that are looked at in the epilogue: on the way from here in the large tiles, whose waves all store at once (2000
  // tokens on V = 50021, K = 512 in bf16 86.3 us, loaded there 88.2), but loaded there in the small ones, which wait for
  // the first operands (48 tokens on V = 16000, K = 4096 20.8 us, from here 21.7).
  Scales<FM, FN> scales;
  constexpr bool kEarly = NT > 256;
  if constexpr (kEarly) scales.load(p, v0, n0);
  const uint32_t lds0 = lds_addr(smem);
  TA ta;
  ta.setup(p.w, vt * BV, p.S);
  TB th;
  th.setup(p.h, tb * BM, p.S);
  int is = 0, is_slot = 0;
  auto issue_next = [&]() {
    if (is >= p.S) return;
    const uint32_t st = lds0 + is_slot * SB;
    ta.issue(st, is);
    th.issue(st + TA::BYTES, is);
    ++is;
    is_slot = is_slot == NS - 1 ? 0 : is_slot + 1;
  };
#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue_next();
  i32x16_t acc[FM][FN];
#pragma unroll
  for (int fm = 0; fm < FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < FN; ++fn)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[fm][fn][r] = 0;
  Ring<NS> ring{NS - 1, p.S};
  ring.template publish_next<L>();
  tile_reduce<int8_t, 32, L>(acc, ta, th, smem, SB, ring, p.S, wv * (BV / WV), wt * (BM / WT), issue_next);  // (two steps a slice)
  stage_barrier();  // every wave has read its last operands: the ring holds the epilogue's rows
  constexpr int kRoom = NS * SB / (WV * WT);
  if constexpr (!kEarly) scales.load(p, v0, n0);
  auto store = [&](auto by) {
    store_tile<Out, FM, FN, kRoom, decltype(by)::value>(p, acc, smem + w * kRoom, s_scale + wv * (BV / WV),
                                                        s_bias + wv * (BV / WV), v0, n0);
  };
  if (scales.far(p.scale)) [[unlikely]]
    store(std::true_type());
  else
    store(std::false_type());
}

template <class Src>
hipError_t quantize_typed(const Src* x, int64_t ld, int64_t R, int64_t K64, char* image, float* scale, int pad,
                          hipStream_t stream) {
  const int K = (int)K64, S = (int)int8_slices(K);
  const int64_t rows = pad ? (R + kInt8Rows - 1) / kInt8Rows * kInt8Rows : R;
  const unsigned many = (unsigned)((rows + kManyRows - 1) / kManyRows);
  // A wave a row where that is one piece for each lane or fills the card with 2048 rows.  (bf16: 1000 rows of 1000 4.2 us,
  // with a workgroup a row 5.2; of 4096 500 rows 8.8 and 5.6, 2048 9.9 and 10.6, 8192 22 and 34.)
  if (K <= 1024)
    int8_quantize_kernel<Src, 64, 1><<<many, 64 * kManyRows, 0, stream>>>(x, ld, R, K, S, image, scale);
  else if (rows < 2048)
    int8_quantize_kernel<Src, 256, 2><<<(unsigned)rows, 256, 0, stream>>>(x, ld, R, K, S, image, scale);
  else if (K <= 4096)
    int8_quantize_kernel<Src, 64, 4><<<many, 64 * kManyRows, 0, stream>>>(x, ld, R, K, S, image, scale);
  else
    int8_quantize_kernel<Src, 64, 8><<<many, 64 * kManyRows, 0, stream>>>(x, ld, R, K, S, image, scale);
  return hipGetLastError();
}

template <class Out, int BV, int BM, int WV, int WT, int NS>
void tile_launch(Int8Params p, hipStream_t stream) {
  p.n_vt = (p.V + BV - 1) / BV;
  p.n_tb = (p.N + BM - 1) / BM;
  int8_tile_kernel<Out, BV, BM, WV, WT, NS><<<(unsigned)(p.n_vt * p.n_tb), 64 * WV * WT, 0, stream>>>(p);
}

// Tiles that fill the card: about one for each of its 256 CUs.
constexpr int64_t kFull = 240;

// Up to 64 tokens reading W bounds a call, at up to 5.6 TB/s, which tiles of 128 x 64 through LDS reach; on few rows the
// kernel without LDS, whose workgroups of 32 rows are more: (K = 4096, V = 16000, 1 token: 11.1 us, tiles 16.0; K = 2560, V =
// 151936, 48 tokens: 99 us, tiles 81.)  The border: 32 tokens take tiles from 240 of them on (V = 30593), more tokens from
// half as many (V = 15297), where both are alike (48 tokens, K = 4096, V = 15400 19.6 us without LDS and 20.2, 16000 19.6 and
// 19.7, 20000 21.6 and 20.5, 28000 28.0 and 24.1; tiles of 64 x 64 18.2 on 16000, 22.1 on 20000, 24.1 on 28000).
// With more tokens the largest tile that fills the
// card (200 tokens, K = 4096: 256 x 256 on V = 128256 142 us and 256 x 128 153; on V = 32000 52 and 37; 128 x 128 on V =
// 16000 24, 256 x 128 28), and of 256 x 256 and 256 x 128 the one with the fewer padded tokens.  With K up to 512, in fp32
// 1024, storing logits takes as long as forming them, and 256 x 128, two to a CU, does one beside the other.  (256 x 256 and
// 256 x 128: 500 tokens on V = 50021, K = 512 in bf16 33.4 and 32.5 us; 8192 on 50048, K = 512 in bf16 323 and 315, in fp32 402
// and 382; 1000 on 32000, K = 1024 in fp32 55.5 and 49.9.  Past the border: 8192 on 50048, K = 1024 in bf16 468 and 465, K = 1536
// 623 and 630, in fp32 701 and 707, but 1000 on 32000, K = 1024 in bf16 44.9 and 43.6, K = 1536 in fp32 69.5 and 64.5.)
template <class Out>
hipError_t logits_typed(Int8Params p, hipStream_t stream) {
  // Logits past the caches where rows are whole lines (a wave writes 256 bytes of each): W and h stay in them.  (8192
  // tokens, K = 4096, V = 128256 3660 -> 3505 us, 100 tokens, K = 2560, V = 151936 102 -> 92; on V = 50021, whose rows
  // share lines, 500 tokens in fp32 55 -> 75.)
  p.lines = reinterpret_cast<uintptr_t>(p.out) % 128 == 0 && (int64_t)p.V * sizeof(Out) % 128 == 0;
  auto tiles = [&](int bv, int bm) { return (int64_t)((p.V + bv - 1) / bv) * ((p.N + bm - 1) / bm); };
  auto padded = [&](int bm) { return (int64_t)((p.N + bm - 1) / bm * bm); };
  const bool stores = p.S * (int)kInt8K <= 256 * (int)sizeof(Out);
  if (p.N <= 32 && tiles(128, 32) < kFull)
    int8_few_kernel<Out, 1, 1, 4><<<(unsigned)((p.V + 31) / 32), 256, 0, stream>>>(p);
  else if (p.N > 32 && p.N <= 64 && tiles(64, 64) < kFull)
    int8_few_kernel<Out, 2, 1, 2><<<(unsigned)((p.V + 31) / 32), 256, 0, stream>>>(p);
  else if (p.N <= 64)
    tile_launch<Out, 128, 64, 2, 2, 4>(p, stream);
  else if (p.N > 128 && !stores && tiles(256, 256) >= kFull && padded(256) <= 1.05 * padded(128))
    tile_launch<Out, 256, 256, 2, 4, 3>(p, stream);
  else if (p.N > 128 && tiles(256, 128) >= kFull)
    tile_launch<Out, 256, 128, 4, 2, 3>(p, stream);
  else if (tiles(128, 128) >= kFull)
    tile_launch<Out, 128, 128, 2, 4, 4>(p, stream);
  else
    tile_launch<Out, 64, 128, 2, 2, 4>(p, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t int8_quantize(int dtype, const void* x, int64_t ld, int64_t R, int64_t K, void* image, float* scale, int pad,
                         hipStream_t stream) {
  if (R == 0) return hipSuccess;
  char* im = static_cast<char*>(image);
  hipError_t e;
  timing_begin(kKindInt8Rows, stream);
  switch (dtype) {
    case kBF16: e = quantize_typed(static_cast<const bf16_t*>(x), ld, R, K, im, scale, pad, stream); break;
    case kF16: e = quantize_typed(static_cast<const f16_t*>(x), ld, R, K, im, scale, pad, stream); break;
    default: e = quantize_typed(static_cast<const float*>(x), ld, R, K, im, scale, pad, stream); break;
  }
  timing_end(kKindInt8Rows, stream);
  return e;
}

hipError_t int8_pack(const void* q, int64_t ld, int64_t R, int64_t K, void* image, hipStream_t stream) {
  if (R == 0) return hipSuccess;
  const int vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 16 == 0;
  const int64_t rows = (R + kInt8Rows - 1) / kInt8Rows * kInt8Rows;
  timing_begin(kKindInt8Rows, stream);
  int8_pack_kernel<<<(unsigned)(rows / 32), 256, 0, stream>>>(static_cast<const int8_t*>(q), ld, R, (int)K,
                                                              (int)int8_slices(K), vec, static_cast<char*>(image));
  timing_end(kKindInt8Rows, stream);
  return hipGetLastError();
}

hipError_t int8_unpack(const void* image, const float* scale, int64_t R, int64_t K, float* out, hipStream_t stream) {
  if (R == 0 || K == 0) return hipSuccess;
  timing_begin(kKindInt8Rows, stream);
  const int pieces = (int)((K + kUnpackK - 1) / kUnpackK);
  int8_unpack_kernel<<<(unsigned)((R + 31) / 32 * pieces), 256, 0, stream>>>(static_cast<const char*>(image), scale, R, (int)K,
                                                                             (int)int8_slices(K), pieces, out);
  timing_end(kKindInt8Rows, stream);
  return hipGetLastError();
}

hipError_t int8_logits(int out_dtype, Int8Params p, hipStream_t stream) {
  if (p.N == 0 || p.V == 0) return hipSuccess;
  hipError_t e;
  timing_begin(kKindInt8, stream);
  switch (out_dtype) {
    case kBF16: e = logits_typed<bf16_t>(p, stream); break;
    case kF16: e = logits_typed<f16_t>(p, stream); break;
    default: e = logits_typed<float>(p, stream); break;
  }
  timing_end(kKindInt8, stream);
  return e;
}

}  // namespace swvr
