// Pieces shared by the attention kernels over the block-scaled cache.
#pragma once

#include "fca_attend_common.h"
#include "fca_block_scales.h"

namespace fca {

// A row whose scores held a NaN has a sum that is none.  The merge drops a partial without a
// log-sum-exp as an empty one; this tag in the row's scale, which points to no second partial, makes
// it give NaN for the row and its log-sum-exp instead.
constexpr int kNanTag = 1;
// Left operand and right operand of the product that finds NaN values a row sees: their product
// overflows, each alone is a bf16 number.
constexpr float kHuge = 0x1p120f;

// 0xff in every byte of a dword of codes that holds a NaN (0x7f or 0xff).
__device__ inline unsigned nan_bytes(unsigned w) {
  const unsigned x = (w & 0x7f7f7f7fu) + 0x01010101u;  // bit 7 of a byte: its magnitude was 0x7f
  return ((x & 0x80808080u) >> 7) * 0xffu;
}
// kHuge where one of eight codes is NaN, 0 elsewhere.
__device__ inline bf16x8 huge_at_nans(i32x2 w) {
  bf16x8 r;
#pragma unroll
  for (int k = 0; k < 8; ++k) r[k] = (__bf16)((((unsigned)w[k >> 2] >> (8 * (k & 3))) & 0x7f) == 0x7f ? kHuge : 0.f);
  return r;
}
// The value the lane 32 away holds, without a trip through LDS.
__device__ inline float other_half(float x) {
  const unsigned u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}
// Codes of tokens 8h..8h+7 for channel block db from the raw V registers of its pair of channel blocks:
// rows of channel blocks 2 * pair and 2 * pair + 1 sit in the lower and upper lane halves.
__device__ inline i32x2 value_codes(i32x4 raw, int db) {
  const auto s0 = __builtin_amdgcn_permlane32_swap((unsigned)raw[0], (unsigned)raw[2], false, false);
  const auto s1 = __builtin_amdgcn_permlane32_swap((unsigned)raw[1], (unsigned)raw[3], false, false);
  return i32x2{(int)s0[db & 1], (int)s1[db & 1]};
}
// The first `n` of the 16 codes of a raw V register (the tokens of one block); n is wave-uniform, so
// the masks are scalar.  Codes behind them are whatever the cache holds past the last token.
__device__ inline i32x4 first_codes(i32x4 raw, int n) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = n - 4 * j;
    raw[j] &= k >= 4 ? -1 : k <= 0 ? 0 : (int)((1u << (8 * k)) - 1);
  }
  return raw;
}
// The same for a lane's own eight codes.
__device__ inline i32x2 first_codes(i32x2 w, int n) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int k = n - 4 * j;
    w[j] &= k >= 4 ? -1 : k <= 0 ? 0 : (int)((1u << (8 * k)) - 1);
  }
  return w;
}
// The codes without those that are NaN; `found` collects where there were any.
template <class V>
__device__ inline V without_nans(V raw, int& found) {
#pragma unroll
  for (int j = 0; j < (int)(sizeof(V) / 4); ++j) {
    const int bad = (int)nan_bytes((unsigned)raw[j]);
    raw[j] &= ~bad;
    found |= bad;
  }
  return raw;
}

// 64-row items (head sizes 64 and 128) and head size 256: fca_attend_block_wide.hip
hipError_t launch_attend_block_wide(const AttendParams& p, const fca_plan& plan, int cus, int max_workgroups, hipStream_t stream);

}  // namespace fca
