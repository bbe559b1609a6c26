// Rows of logits: keys that order them, and moves between the lanes of a wave (sampling, beam selection).
#pragma once
#include "common.hpp"

namespace swvr {

typedef unsigned long long u64;

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

// A token whose place in the order is its key and then its index, as one number: larger is earlier; 0: nothing.
__device__ __forceinline__ u64 place_of(uint32_t key, int64_t i) {
  return key == 0 ? 0 : (u64)key << 32 | (uint32_t)~(uint32_t)i;
}
__device__ __forceinline__ uint32_t key_at(u64 place) { return (uint32_t)(place >> 32); }
__device__ __forceinline__ int64_t index_at(u64 place) { return (int64_t)(uint32_t)~(uint32_t)place; }

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

}  // namespace swvr
