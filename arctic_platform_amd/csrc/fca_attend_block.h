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

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
// 8 e4m3 codes -> 8 halves (every e4m3 value is one, so the conversion is exact).
__device__ inline f16x8 fp8x8_to_f16(i32x2 w) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

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

// ---- softmax of one query row (a lane and the one 32 away hold one) ----------------------------
// The value product takes the weights p * s_v as halves: 11 significant bits where bf16 has 8, at the
// same rate of the matrix cores.  What is left of the error of a bf16 output is the rounding of the
// output: 0.0015 to 0.0020 relative to the definition in 64 bits over the measured cases, within a
// twentieth of what fp32 weights give on the same inputs (bf16 weights: 0.0019 to 0.0022, up to 1.35 times).  A half spans 2^-24 to 2^15, so the weights have a reference
// of their own next to that of the exponentials: the largest log2(p) + log2(s_v) the row has met.
// The largest weight is then about 2^kWeightBits; one 2^-21 of it still has 11 bits, and what is lost
// of a smaller one is below 2^-32 of the largest, whatever the scales of the blocks are.  Measured
// against bf16 weights with one reference: 0 to 4 % of a call (verify steps 52.4 -> 54.7 us the most).
constexpr float kWeightBits = 7.f;  // + kRescaleSlack = 15: a half ends at 65504
struct RowState {
  float m;  // reference of the scaled scores (log2 domain)
  float u;  // that of the weights: largest (score - m) + log2(V scale).  (Relative to m, and from the fused
            // multiply-add the exponentials take: scores far beyond 2^24 would leave nothing of a V scale's log2
            // added to them, and their rounding alone moves the exponent of a weight by more than a half holds.)
  float g;  // 2^(kWeightBits - u): weight = exp2(score - m) * V scale * g
  float l;  // running sum of exp2(score - m)
};
__device__ inline RowState empty_row() { return RowState{-INFINITY, -INFINITY, 1.f, 0.f}; }
// log2 of a V scale, kept from where the writer's scales begin (g stays finite; a weight under a smaller scale,
// in a table of somebody else's, has fewer bits).
__device__ inline float scale_log2(float vs) { return fmaxf(fast_log2(vs), (float)(kScaleExpMin - 127)); }

// Scores of a tile -> weights, register r holding token 16 * (r / 8) + 8 * h + r % 8 of the tile; ks, vs, lv:
// K scale (log2 domain), V scale and its log2 of the tile's two blocks.  RAGGED: registers of tokens from
// `lim` on (counted from 8 * h) are masked.
template <bool RAGGED, int NDB>
__device__ inline void weigh_tile(RowState& row, bool first, f32x16 sr, const float (&ks)[2], const float (&vs)[2], const float (&lv)[2], int lim,
                                  f32x16 (&acc)[NDB], f16x8 (&weights)[2]) {
  if constexpr (RAGGED) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (16 * (r >> 3) + (r & 7) >= lim) sr[r] = -INFINITY;
  }
  float mx[2];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    mx[blk] = sr[8 * blk];
#pragma unroll
    for (int r = 1; r < 8; ++r) mx[blk] = fmaxf(mx[blk], sr[8 * blk + r]);
  }
  // (the scales are positive, so the maximum of the scaled scores is a scaled maximum)
  float mtile = fmaxf(mx[0] * ks[0], mx[1] * ks[1]);
  mtile = fmaxf(mtile, other_half(mtile));
  auto largest_weight = [&]() {
    const float x = fmaxf(__builtin_fmaf(mx[0], ks[0], -row.m) + lv[0], __builtin_fmaf(mx[1], ks[1], -row.m) + lv[1]);
    return fmaxf(x, other_half(x));
  };
  // The references move (and sum and accumulators are rescaled) only when a maximum rises more than
  // kRescaleSlack above its own.  (That a lane looks at its half of the tile's weights first, and at the
  // other's where it has to, costs the wide kernels scratch: verify steps 69 us instead of 54.7.)
  if (first) row.m = mtile;
  float utile = largest_weight();
  if (first) row.u = utile, row.g = fast_exp2(kWeightBits - utile);
  if (__ballot(mtile > row.m + kRescaleSlack || utile > row.u + kRescaleSlack) != 0) {
    const float drop = row.m - fmaxf(row.m, mtile);
    row.m = fmaxf(row.m, mtile);
    utile = largest_weight();
    const float u_new = fmaxf(row.u + drop, utile);
    const float alpha = fast_exp2(row.u + drop - u_new);
    row.l *= fast_exp2(drop);
    row.u = u_new;
    row.g = fast_exp2(kWeightBits - u_new);
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
  }
  const float factor[2] = {vs[0] * row.g, vs[1] * row.g};
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float e = fast_exp2(__builtin_fmaf(sr[r], ks[r >> 3], -row.m));
    // (by its place: minus infinity may be a score too, and times a scale of zero it is no number)
    if (RAGGED && 16 * (r >> 3) + (r & 7) >= lim) e = 0.f;
    sum += e;
    weights[r >> 3][r & 7] = (_Float16)(e * factor[r >> 3]);
  }
  row.l += sum;
}

// 64-row items (head sizes 64 and 128) and head size 256: fca_attend_block_wide.hip
hipError_t launch_attend_block_wide(const AttendParams& p, const fca_plan& plan, int cus, int max_workgroups, hipStream_t stream);

}  // namespace fca
