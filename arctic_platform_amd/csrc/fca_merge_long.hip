// Log-sum-exp merge of rows with many partials (long sequences cut into many chunks): one workgroup
// per (sequence, query head) row.
//
// The merge of fca_merge.hip gives a row at most one wave; with the 128 partials of a sequence of
// 131072 tokens that is eight round trips to memory one after the other, and a single sequence of 32
// query heads occupies 8 of 256 CUs (9.3 us, against 44 us of the attention in front of it).
// Here 2048 / D groups of D / 8 lanes take every (2048 / D)-th partial of the row each, four at a
// time, all loads of a batch in flight together, and combine in registers and LDS: one round trip for
// up to 64 partials at D = 128 (4.9 us for those 128).  How many partials a row has is known here, not
// where the kernel is chosen: a row that one wave covers in one batch is left to one wave (2.8 us at 16
// partials).  Partial rows, tags and NaN rules are those of fca_merge.hip, to
// which the block-scaled cache adds that a second partial carries a tag of its own where its row is
// no number (fca_attend_block.h).
#include <hip/hip_bf16.h>

#include "fca_block_scales.h"

namespace fca {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));

struct Running {  // maximum, sum of weights, weighted sum of eight channels
  float m, wsum, acc[8];
};
__device__ inline void add_partial(Running& r, float l, float scale, const half8& o) {
  const bool live = l > -INFINITY;  // (an empty partial has weight 0 whatever its output holds)
  const float m_new = fmaxf(r.m, l);
  const float keep = r.m > -INFINITY ? __expf(r.m - m_new) : 0.f;
  const float w = live ? __expf(l - m_new) : 0.f;
  r.wsum = r.wsum * keep + w;
  const float ws = w * scale;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.acc[e] = r.acc[e] * keep + (live ? ws * (float)o[e] : 0.f);
  r.m = m_new;
}
__device__ inline void add_running(Running& r, const Running& o) {
  const float m_new = fmaxf(r.m, o.m);
  const float keep = r.m > -INFINITY ? __expf(r.m - m_new) : 0.f;
  const float take = o.m > -INFINITY ? __expf(o.m - m_new) : 0.f;
  r.wsum = r.wsum * keep + o.wsum * take;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.acc[e] = r.acc[e] * keep + o.acc[e] * take;
  r.m = m_new;
}

template <int D>
__global__ __launch_bounds__(256) void fca_merge_long_kernel(MergeParams p) {
  constexpr int LPS = D / 8;          // lanes per share of a row
  constexpr int B = 4;
  constexpr int WAVE_SHARES = 64 / LPS;
  __shared__ Running part[4][LPS];
  __shared__ int part_stray[4];
  const int row = blockIdx.x, s = row / p.num_q_heads, hq = row - s * p.num_q_heads;
  const int tid = threadIdx.x, sub = tid % LPS, share = tid / LPS, wave = tid >> 6, lane = tid & 63;
  const int np = p.seq_npart[s];
  // a row that one wave covers in one batch is that wave's alone
  const bool one_wave = np <= B * WAVE_SHARES;
  if (one_wave && wave != 0) return;
  const int shares = one_wave ? WAVE_SHARES : 4 * WAVE_SHARES;
  const int64_t base = (int64_t)s * p.max_partials;
  const _Float16* rows = static_cast<const _Float16*>(p.partial_out);
  const float2v* lse_scale = reinterpret_cast<const float2v*>(p.partial_lse);
  Running r;
  r.m = -INFINITY, r.wsum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.acc[e] = 0.f;
  int stray = 0;
  for (int i0 = share; i0 < np; i0 += B * shares) {
    float2v ls[B];
    half8 o[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {  // (past the row's last partial: that one again, at weight 0)
      const int64_t pr = (base + min(i0 + j * shares, np - 1)) * p.num_q_heads + hq;
      ls[j] = __builtin_nontemporal_load(lse_scale + pr);
      o[j] = __builtin_nontemporal_load(reinterpret_cast<const half8*>(rows + pr * D + sub * 8));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (i0 + j * shares >= np) ls[j] = float2v{-INFINITY, 1.f};
      const unsigned tag = __float_as_uint(ls[j][1]) & 0x007fffffu;
      add_partial(r, ls[j][0], __uint_as_float(__float_as_uint(ls[j][1]) & 0xff800000u), o[j]);
      if (tag == 0) continue;
      // a second partial of the same chunk, or, where the tag points to none, a row that is no number
      if (tag < 32 || (int64_t)tag - 32 >= p.coop_rows) {
        stray = 1;
        continue;
      }
      const int64_t br = p.coop_row0 + tag - 32;
      const float2v bls = lse_scale[br];
      if ((__float_as_uint(bls[1]) & 0x007fffffu) != 0) stray = 1;
      add_partial(r, bls[0], __uint_as_float(__float_as_uint(bls[1]) & 0xff800000u), *reinterpret_cast<const half8*>(rows + br * D + sub * 8));
    }
  }
  // the shares of a wave, then the waves
#pragma unroll
  for (int off = LPS; off < 64; off <<= 1) {
    Running x;
    x.m = __shfl_xor(r.m, off), x.wsum = __shfl_xor(r.wsum, off);
#pragma unroll
    for (int e = 0; e < 8; ++e) x.acc[e] = __shfl_xor(r.acc[e], off);
    stray |= __shfl_xor(stray, off);
    add_running(r, x);
  }
  if (!one_wave) {
    if (lane < LPS) part[wave][lane] = r;
    if (lane == 0) part_stray[wave] = stray;
    __syncthreads();
  }
  if (tid >= LPS) return;
  if (!one_wave) {
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      add_running(r, part[w][sub]);
      stray |= part_stray[w];
    }
  }
  // input the builder had to clamp makes every output NaN, as in fca_merge.hip
  const bool flagged = p.header[H_ERROR] != 0 || stray != 0;
  const float inv = flagged ? __builtin_nanf("") : (r.wsum > 0.f ? 1.f / r.wsum : 0.f);
  const int64_t o = (int64_t)s * p.out_seq_stride + (int64_t)hq * p.out_head_stride + sub * 8;
  if (p.out_dtype == FCA_F32) {
    float* dst = reinterpret_cast<float*>(p.out) + o;
    if (p.vector_out) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(r.acc[0] * inv, r.acc[1] * inv, r.acc[2] * inv, r.acc[3] * inv);
      reinterpret_cast<float4*>(dst)[1] = make_float4(r.acc[4] * inv, r.acc[5] * inv, r.acc[6] * inv, r.acc[7] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = r.acc[e] * inv;
    }
  } else {
    __hip_bfloat16* dst = reinterpret_cast<__hip_bfloat16*>(p.out) + o;
    union {
      __hip_bfloat16 h[8];
      uint4 u;
    } pack;
#pragma unroll
    for (int e = 0; e < 8; ++e) pack.h[e] = __float2bfloat16(r.acc[e] * inv);
    if (p.vector_out) {
      *reinterpret_cast<uint4*>(dst) = pack.u;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = pack.h[e];
    }
  }
  if (p.lse && sub == 0) p.lse[row] = flagged ? __builtin_nanf("") : (r.wsum > 0.f ? r.m + __logf(r.wsum) : -INFINITY);
}

hipError_t launch_merge_long(const MergeParams& p, hipStream_t stream) {
  const unsigned rows = (unsigned)p.num_seqs * (unsigned)p.num_q_heads;
  if (rows == 0) return hipSuccess;
  if (p.head_dim == 64)
    hipLaunchKernelGGL(fca_merge_long_kernel<64>, dim3(rows), dim3(256), 0, stream, p);
  else if (p.head_dim == 128)
    hipLaunchKernelGGL(fca_merge_long_kernel<128>, dim3(rows), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(fca_merge_long_kernel<256>, dim3(rows), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fca
