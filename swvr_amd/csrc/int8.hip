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

// 16 consecutive values of a row from k on, 0 past K; vec: 16-byte aligned rows.
template <class Src>
__device__ __forceinline__ void load16(const Src* row, int k, int K, bool vec, float (&v)[16]) {
  if (vec && k + 16 <= K) {
    constexpr int CE = 16 / (int)sizeof(Src);
    struct alignas(16) X {
      Src v[CE];
    };
#pragma unroll
    for (int j = 0; j < 16 / CE; ++j) {
      const X x = *reinterpret_cast<const X*>(row + k + j * CE);
#pragma unroll
      for (int i = 0; i < CE; ++i) v[j * CE + i] = (float)x.v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = k + i < K ? (float)row[k + i] : 0.f;
  }
}

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

// TPR threads a row: 8 for many rows, whose 16-byte chunks then go out as 128-byte runs; a workgroup for few.
template <class Src, int TPR>
__global__ __launch_bounds__(256) void int8_quantize_kernel(const Src* __restrict__ x, int64_t ld, int64_t R, int K, int S,
                                                            int vec, char* __restrict__ image, float* __restrict__ scale) {
  __shared__ uint32_t s_max[4];
  const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int j = threadIdx.x % TPR;
  const Src* row = x + r * ld;
  // the largest magnitude by its bits: an infinity or a NaN is larger than any number
  uint32_t m = 0;
  if (r < R)
    for (int k = j * 16; k < K; k += TPR * 16) {
      float v[16];
      load16(row, k, K, vec != 0, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        m = b > m ? b : m;
      }
    }
#pragma unroll
  for (int o = 1; o < (TPR < 64 ? TPR : 64); o <<= 1) {
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
  char* out = image + (r >> 5) * S * kInt8Block + (r & 31) * 16;
  for (int k = j * 16; k < S * 64; k += TPR * 16) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (r < R && fine && k < K) {
      float v[16];
      load16(row, k, K, vec != 0, v);
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i / 4] |= (uint32_t)(quantize(v[i], s, inv, half) & 255) << (8 * (i % 4));
    }
    *reinterpret_cast<uint4*>(out + (int64_t)(k >> 4) * 512) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows of integers [R][ld] into an image, 8 threads a row.
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

// The values that an image stands for, in fp32 [R][K], 8 threads a row.
__global__ __launch_bounds__(256) void int8_unpack_kernel(const char* __restrict__ image, const float* __restrict__ scale,
                                                          int64_t R, int K, int S, float* __restrict__ out) {
  const int64_t r = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  if (r >= R) return;
  const char* in = image + (r >> 5) * S * kInt8Block + (r & 31) * 16;
  const float s = scale[r];
  float* row = out + r * K;
  for (int k = (threadIdx.x % 8) * 16; k < K; k += 128) {
    const uint4 w = *reinterpret_cast<const uint4*>(in + (int64_t)(k >> 4) * 512);
    int8_t b[16];
    __builtin_memcpy(b, &w, 16);
    if (K % 4 == 0 && k + 16 <= K) {
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(row + k + i) = make_float4(b[i] * s, b[i + 1] * s, b[i + 2] * s, b[i + 3] * s);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < K) row[k + i] = b[i] * s;
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

// Up to 32 NB tokens: bound by reading W's integers once.  A workgroup takes 32 G of W's rows, its four waves a
// quarter of the reduction each, operands straight from memory; the quarters are added in LDS.
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
    if (v < p.V) out[(int64_t)n * p.V + v] = (Out)fmaf((float)sum, p.scale * p.h_scale[n] * sw, bias);
  }
}

// 16 bytes of logits at any element.
template <class Out>
struct __attribute__((packed, aligned(sizeof(Out)))) OutChunk {
  Out v[16 / sizeof(Out)];
};

// A wave's 32 FM vocabulary rows (from v0) x 32 FN tokens (from n0), through `room` (LDS of this wave, 8704 bytes): a
// lane holds 4 rows of a token, and goes out with 16 bytes of a token's 256.
template <class Out, int FM, int FN>
__device__ __forceinline__ void store_tile(const Int8Params& p, const i32x16_t (&acc)[FM][FN], char* room,
                                           const float* scale, const float* bias, int v0, int n0) {
  constexpr int E = (int)sizeof(Out), FP = 8 / E, kPitch = 256 + 16;  // FP: blocks of 32 rows in 256 bytes
  static_assert(FM % FP == 0, "whole pieces");
  struct alignas(4 * E) Four {
    Out v[4];
  };
  const int lane = lane_id();
#pragma unroll
  for (int fn = 0; fn < FN; ++fn) {
    const int nb = n0 + fn * 32, n = nb + (lane & 31);
    const float sh = n < p.N ? p.scale * p.h_scale[n] : 0.f;
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
          for (int i = 0; i < 4; ++i) y.v[i] = (Out)fmaf((float)acc[f0 + f][fn][4 * g + i], sh * sws[i], bs[i]);
          *reinterpret_cast<Four*>(room + (lane & 31) * kPitch + c * E) = y;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = i * 4 + lane / 16, at = (lane % 16) * 16;
        const int v = v0 + f0 * 32 + at / E;
        const OutChunk<Out> y = *reinterpret_cast<const OutChunk<Out>*>(__builtin_assume_aligned(room + t * kPitch + at, 16));
        if (nb + t >= p.N) continue;
        Out* const to = static_cast<Out*>(p.out) + (int64_t)(nb + t) * p.V + v;
        if (v + 16 / E <= p.V) {
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

// Many tokens: 256 x 256 tiles of 8 waves, the readout's reduction loop (tile_reduce) on integer operands.
constexpr int kBV = 256, kBM = 256, kTileThreads = 512;
template <class Out>
__global__ __launch_bounds__(kTileThreads) void int8_tile_kernel(Int8Params p) {
  constexpr int NS = 4, FM = 4, FN = 2;
  typedef I8Tile<kBV, kTileThreads> TA;
  typedef I8Tile<kBM, kTileThreads> TB;
  constexpr int SB = TA::BYTES + TB::BYTES, L = TA::NI + TB::NI;
  __shared__ __attribute__((aligned(1024))) char smem[NS * SB];
  __shared__ __attribute__((aligned(16))) float s_scale[kBV], s_bias[kBV];
  const int w = wave_id(), wv = w >> 2, wt = w & 3;
  int vt, tb;
  grouped_tile(blockIdx.x, p.n_vt, p.n_tb, &vt, &tb);
  if (threadIdx.x < kBV) {
    s_scale[threadIdx.x] = wscale_at(p, vt * kBV + (int)threadIdx.x);
    s_bias[threadIdx.x] = bias_at(p, vt * kBV + (int)threadIdx.x);
  }
  const uint32_t lds0 = lds_addr(smem);
  TA ta;
  ta.setup(p.w, vt * kBV, p.S);
  TB th;
  th.setup(p.h, tb * kBM, p.S);
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
  tile_reduce<int8_t, 32, L>(acc, ta, th, smem, SB, ring, p.S, wv * 128, wt * 64, issue_next);  // (two steps a slice)
  stage_barrier();  // every wave has read its last operands: the ring holds the epilogue's rows
  store_tile<Out, FM, FN>(p, acc, smem + w * (NS * SB / 8), s_scale + wv * 128, s_bias + wv * 128, vt * kBV + wv * 128,
                          tb * kBM + wt * 64);
}

template <class Src>
hipError_t quantize_typed(const Src* x, int64_t ld, int64_t R, int64_t K, char* image, float* scale, int pad,
                          hipStream_t stream) {
  const int S = (int)int8_slices(K);
  const int vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (ld * (int64_t)sizeof(Src)) % 16 == 0;
  const int64_t rows = pad ? (R + kInt8Rows - 1) / kInt8Rows * kInt8Rows : R;
  if (R < 8192)
    int8_quantize_kernel<Src, 256><<<(unsigned)rows, 256, 0, stream>>>(x, ld, R, (int)K, S, vec, image, scale);
  else
    int8_quantize_kernel<Src, 8><<<(unsigned)((rows + 31) / 32), 256, 0, stream>>>(x, ld, R, (int)K, S, vec, image, scale);
  return hipGetLastError();
}

template <class Out>
hipError_t logits_typed(Int8Params p, hipStream_t stream) {
  if (p.N <= 32) {
    int8_few_kernel<Out, 1, 1, 4><<<(unsigned)((p.V + 31) / 32), 256, 0, stream>>>(p);
  } else if (p.N <= 64) {
    int8_few_kernel<Out, 2, 1, 2><<<(unsigned)((p.V + 31) / 32), 256, 0, stream>>>(p);
  } else {
    p.n_vt = (p.V + kBV - 1) / kBV;
    p.n_tb = (p.N + kBM - 1) / kBM;
    int8_tile_kernel<Out><<<(unsigned)(p.n_vt * p.n_tb), kTileThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t int8_quantize(int dtype, const void* x, int64_t ld, int64_t R, int64_t K, void* image, float* scale, int pad,
                         hipStream_t stream) {
  if (R == 0) return hipSuccess;
  char* im = static_cast<char*>(image);
  hipError_t e;
  timing_begin(kKindQuant, stream);
  switch (dtype) {
    case kBF16: e = quantize_typed(static_cast<const bf16_t*>(x), ld, R, K, im, scale, pad, stream); break;
    case kF16: e = quantize_typed(static_cast<const f16_t*>(x), ld, R, K, im, scale, pad, stream); break;
    default: e = quantize_typed(static_cast<const float*>(x), ld, R, K, im, scale, pad, stream); break;
  }
  timing_end(kKindQuant, stream);
  return e;
}

hipError_t int8_pack(const void* q, int64_t ld, int64_t R, int64_t K, void* image, hipStream_t stream) {
  if (R == 0) return hipSuccess;
  const int vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 16 == 0;
  const int64_t rows = (R + kInt8Rows - 1) / kInt8Rows * kInt8Rows;
  timing_begin(kKindQuant, stream);
  int8_pack_kernel<<<(unsigned)(rows / 32), 256, 0, stream>>>(static_cast<const int8_t*>(q), ld, R, (int)K,
                                                              (int)int8_slices(K), vec, static_cast<char*>(image));
  timing_end(kKindQuant, stream);
  return hipGetLastError();
}

hipError_t int8_unpack(const void* image, const float* scale, int64_t R, int64_t K, float* out, hipStream_t stream) {
  if (R == 0 || K == 0) return hipSuccess;
  timing_begin(kKindQuant, stream);
  int8_unpack_kernel<<<(unsigned)((R + 31) / 32), 256, 0, stream>>>(static_cast<const char*>(image), scale, R, (int)K,
                                                                    (int)int8_slices(K), out);
  timing_end(kKindQuant, stream);
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
