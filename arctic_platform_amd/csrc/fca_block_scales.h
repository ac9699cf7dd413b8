// The block-scaled 8-bit cache: e4m3 codes in the tile order of every other fp8 cache, with one
// fp32 scale per (block of 16 tokens, KV head) and plane in a table [num_blocks][Hkv][2] (K's scale,
// V's scale); a code c stands for c * scale.  Pieces shared by its writer, its reader and the
// attention kernels.
#pragma once

#include "fca_common.h"

namespace fca {

constexpr float kE4m3Max = 448.f;
// The writer's scales are powers of two between 2^-100 and 2^120: dividing by one is exact, so the
// only rounding of a stored value is the one to e4m3, and codes that move to a larger scale of
// their block (a later token of the block needs it) move without a rounding as long as they stay
// above the subnormals.  e4m3 is a floating-point format, so a scale between two powers of two
// would gain no precision, only up to one binade at the lower end of its 18.  The lower bound keeps
// 1 / scale finite and a block of zeros usable; the upper one is past what the largest bf16 needs.
constexpr int kScaleExpMin = 127 - 100, kScaleExpMax = 127 + 120;  // biased exponents

__host__ __device__ inline uint32_t float_bits(float x) { return __builtin_bit_cast(uint32_t, x); }
__host__ __device__ inline float bits_float(uint32_t x) { return __builtin_bit_cast(float, x); }

// Biased exponent of the smallest power of two s with x <= s, within the bounds (x >= 0, finite).
__host__ __device__ inline int scale_exp_above(float x) {
  const uint32_t b = float_bits(x);
  const int e = (int)(b >> 23) + ((b & 0x007fffffu) != 0 ? 1 : 0);
  return e < kScaleExpMin ? kScaleExpMin : e > kScaleExpMax ? kScaleExpMax : e;
}
// The same for the smallest power of two s with amax <= 448 s: 448 = 1.75 * 2^8.
__host__ __device__ inline int scale_exp_for(float amax) {
  const uint32_t b = float_bits(amax);
  const int e = (int)(b >> 23) - 8 + ((b & 0x007fffffu) > 0x00600000u ? 1 : 0);
  return e < kScaleExpMin ? kScaleExpMin : e > kScaleExpMax ? kScaleExpMax : e;
}

// tokens of one append call (every workgroup looks at all their slots, with 32-bit indices)
constexpr int32_t kAppendMostTokens = 1 << 30;

struct BlockCacheParams {
  const void* key;  // bf16 [T, Hkv, D]; written by the reader
  const void* value;
  int64_t token_stride, head_stride;  // elements
  const int64_t* slot_mapping;        // [T]
  void* k_cache;
  void* v_cache;
  int64_t cache_block_stride, cache_head_stride;  // elements = bytes
  float* scales;                                  // [num_blocks, Hkv, 2]
  int64_t num_blocks;
  int32_t num_tokens, num_kv_heads, head_dim;
};
hipError_t launch_append_block(const BlockCacheParams& p, hipStream_t stream);
hipError_t launch_gather_block(const BlockCacheParams& p, hipStream_t stream);
hipError_t launch_merge_long(const MergeParams& p, hipStream_t stream);
hipError_t launch_attend_block(const AttendParams& p, const fca_plan& plan, int max_workgroups, hipStream_t stream);

}  // namespace fca
