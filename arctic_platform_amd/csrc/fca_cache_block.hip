// Writer and reader of the block-scaled 8-bit cache (fca_block_scales.h).
//
// Writing.  For a block b, KV head h and plane (K or V) that a call touches, with a = the largest
// finite magnitude among the call's tokens in b:
//   need   = smallest power of two s with a <= 448 s
//   old    = nothing if a token of the call has offset 0 (it begins the block), else the block's scale
//   scale' = max(old, need)
//   codes of the call's tokens = e4m3(x / scale'), nearest, ties to even, saturating; NaN stays NaN
//   where scale' > old, the codes of the other tokens become e4m3(c * old / scale')
// All tokens of a call that fall into one block are handled by the same workgroup, so the scale is
// a maximum over all of them and nothing depends on the order of workgroups: no atomics on global
// memory, no workspace, one launch.  Of two tokens with one slot the later one is written.
//
// Memory-bound: rows in as bf16, codes out.  A wave holds one tile of one plane (16 tokens x D
// codes) in registers: of K a lane takes the 16-byte units (slice of 16 channels, token) with
// token = lane % 16, of V whole channels (16 bytes = their 16 tokens), so both leave as 16-byte
// stores that together cover whole lines, and the maximum is one wave-wide reduction away.
#include <hip/hip_bf16.h>

#include "fca_block_scales.h"

namespace fca {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

__device__ inline float bf16_float(unsigned short x) { return __uint_as_float((unsigned)x << 16); }

__device__ inline unsigned e4m3_code(float x) {
  // saturate (clamp, then round to nearest even); NaN is stored as the canonical 0x7f
  if (x != x) return 0x7f;
  x = fminf(fmaxf(x, -kE4m3Max), kE4m3Max);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xff;
}
// One byte of a dword of codes, scaled and rounded again.
__device__ inline unsigned rescaled_code(unsigned codes, int byte, float ratio) {
  return e4m3_code(__builtin_amdgcn_cvt_f32_fp8((int)(codes >> (8 * byte)), 0) * ratio);
}

__device__ inline float finite_max(float m, unsigned short x) {
  const unsigned short a = x & 0x7fff;
  return a < 0x7f80 ? fmaxf(m, bf16_float(a)) : m;
}

// The scale of one (block, head, plane): what it was, what it becomes.
struct ScaleStep {
  float inv;    // 1 / new scale
  float ratio;  // old / new, for the codes that stay
  bool grown;   // codes that stay have to be rescaled
};
__device__ inline ScaleStep step_scale(float* at, float amax, bool begins, int lane) {
  const float was = *at;  // (every lane has it before the reduction, lane 0 writes behind it)
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
  // (a scale that is no positive finite number, of a block nothing has begun, counts for nothing)
  const bool has_old = !begins && was > 0.f && was < INFINITY;
  int e = scale_exp_for(amax);
  if (has_old) {
    const int eo = scale_exp_above(was);  // (a caller's own scale that is no power of two is raised to one)
    e = e > eo ? e : eo;
  }
  const float scale = __uint_as_float((unsigned)e << 23);
  ScaleStep s;
  s.inv = __uint_as_float((unsigned)(254 - e) << 23);
  s.ratio = was * s.inv;
  s.grown = has_old && scale != was;
  if (lane == 0 && scale != was) *at = scale;
  return s;
}

template <int D>
__device__ inline void append_k_tile(const BlockCacheParams& p, const int* win, int64_t blk, int h, int lane) {
  constexpr int U = D / 64;  // 16-byte units of the tile per lane
  const int tok = lane & 15;
  const int t = win[tok];
  char* tile = static_cast<char*>(p.k_cache) + blk * p.cache_block_stride + h * p.cache_head_stride;
  const unsigned short* row = static_cast<const unsigned short*>(p.key) + (int64_t)t * p.token_stride + (int64_t)h * p.head_stride;
  union {
    int4 raw[2];
    unsigned short x[16];
  } in[U];
  union Codes {
    int4 raw;
    unsigned w[4];
  } out[U];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = (lane >> 4) + 4 * i;
    if (t >= 0) {
      in[i].raw[0] = *reinterpret_cast<const int4*>(row + 16 * c);
      in[i].raw[1] = *reinterpret_cast<const int4*>(row + 16 * c + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = finite_max(amax, in[i].x[e]);
    } else {
      out[i].raw = *reinterpret_cast<const int4*>(tile + (c * kBlock + tok) * 16);
    }
  }
  const ScaleStep s = step_scale(p.scales + (blk * p.num_kv_heads + h) * 2, amax, win[0] >= 0, lane);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = (lane >> 4) + 4 * i;
    if (t < 0 && !s.grown) continue;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      unsigned q = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q |= (t >= 0 ? e4m3_code(bf16_float(in[i].x[4 * d + e]) * s.inv) : rescaled_code(out[i].w[d], e, s.ratio)) << (8 * e);
      out[i].w[d] = q;
    }
    *reinterpret_cast<int4*>(tile + (c * kBlock + tok) * 16) = out[i].raw;
  }
}

template <int D>
__device__ inline void append_v_tile(const BlockCacheParams& p, const int* win, int64_t blk, int h, int lane) {
  constexpr int CH = D / 64;  // adjacent channels per lane
  char* tile = static_cast<char*>(p.v_cache) + blk * p.cache_block_stride + h * p.cache_head_stride + lane * CH * kBlock;
  struct alignas(2 * CH) Piece {
    unsigned short x[CH];
  } in[kBlock];
  union Codes {
    int4 raw;
    unsigned w[4];
  } out[CH];
  float amax = 0.f;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) out[ch].raw = *reinterpret_cast<const int4*>(tile + ch * kBlock);
  unsigned live = 0;
#pragma unroll
  for (int k = 0; k < kBlock; ++k) {
    const int t = __builtin_amdgcn_readfirstlane(win[k]);
    if (t >= 0) {
      live |= 1u << k;
      in[k] = *reinterpret_cast<const Piece*>(static_cast<const unsigned short*>(p.value) + (int64_t)t * p.token_stride +
                                              (int64_t)h * p.head_stride + lane * CH);
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) amax = finite_max(amax, in[k].x[ch]);
    }
  }
  const ScaleStep s = step_scale(p.scales + (blk * p.num_kv_heads + h) * 2 + 1, amax, win[0] >= 0, lane);
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      unsigned q = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 4 * d + e;
        const unsigned kept = s.grown ? rescaled_code(out[ch].w[d], e, s.ratio) : (out[ch].w[d] >> (8 * e)) & 0xff;
        q |= ((live >> k) & 1 ? e4m3_code(bf16_float(in[k].x[ch]) * s.inv) : kept) << (8 * e);
      }
      out[ch].w[d] = q;
    }
    *reinterpret_cast<int4*>(tile + ch * kBlock) = out[ch].raw;
  }
}

// One workgroup per token of the call; the first token of a block in the call owns the block.
template <int D>
__global__ __launch_bounds__(256) void fca_append_block_kernel(BlockCacheParams p) {
  __shared__ int win[kBlock];  // the call's token at every offset of the block, -1 = none
  __shared__ int foreign;
  const int t0 = blockIdx.x, tid = threadIdx.x;
  const int64_t slot = p.slot_mapping[t0];
  if (slot < 0 || slot >= p.num_blocks * kBlock) return;
  const int64_t blk = slot / kBlock;
  if (tid < kBlock) win[tid] = -1;
  if (tid == 0) foreign = 0;
  __syncthreads();
  for (int t = tid; t < p.num_tokens; t += 256) {
    const int64_t s = p.slot_mapping[t];
    if (s < 0 || s / kBlock != blk) continue;
    if (t < t0) foreign = 1;
    atomicMax(&win[s % kBlock], t);
  }
  __syncthreads();
  if (foreign) return;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  for (int j = wave; j < 2 * p.num_kv_heads; j += 4) {
    if (j & 1)
      append_v_tile<D>(p, win, blk, j >> 1, lane);
    else
      append_k_tile<D>(p, win, blk, j >> 1, lane);
  }
}

// Reading back: row t = codes at slot_mapping[t] times their block's scales, rounded to bf16 (exact
// for the writer's scales, short of bf16's own range); a negative slot, or one past the cache, gives
// zeros.  A wave takes 16 tokens of one head and plane.
template <int D>
__global__ __launch_bounds__(256) void fca_gather_block_kernel(BlockCacheParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t task = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = task / (2 * p.num_kv_heads);
  const int j = (int)(task - group * 2 * p.num_kv_heads), h = j >> 1;
  const int64_t t0 = group * 16;
  if (t0 >= p.num_tokens) return;
  const int64_t end = p.num_blocks * kBlock;
  const int64_t t = t0 + (lane & 15);
  int64_t slot = t < p.num_tokens ? p.slot_mapping[t] : -1;
  if (slot >= end) slot = -1;
  const int64_t blk = slot < 0 ? 0 : slot / kBlock;
  const int off = slot < 0 ? 0 : (int)(slot % kBlock);
  const float scale = slot < 0 ? 0.f : p.scales[(blk * p.num_kv_heads + h) * 2 + (j & 1)];
  if ((j & 1) == 0) {
    constexpr int U = D / 64;
    if (t >= p.num_tokens) return;
    const char* tile = static_cast<const char*>(p.k_cache) + blk * p.cache_block_stride + h * p.cache_head_stride;
    __hip_bfloat16* row = static_cast<__hip_bfloat16*>(const_cast<void*>(p.key)) + t * p.token_stride + (int64_t)h * p.head_stride;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = (lane >> 4) + 4 * i;
      union {
        int4 raw;
        unsigned w[4];
      } q;
      union {
        int4 raw[2];
        __hip_bfloat16 x[16];
      } o;
      if (slot >= 0) {
        q.raw = *reinterpret_cast<const int4*>(tile + (c * kBlock + off) * 16);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o.x[e] = __float2bfloat16(__builtin_amdgcn_cvt_f32_fp8((int)(q.w[e >> 2] >> (8 * (e & 3))), 0) * scale);
      } else {
        o.raw[0] = o.raw[1] = make_int4(0, 0, 0, 0);
      }
      reinterpret_cast<int4*>(row + 16 * c)[0] = o.raw[0];
      reinterpret_cast<int4*>(row + 16 * c)[1] = o.raw[1];
    }
  } else {
    constexpr int CH = D / 64;
    struct alignas(2 * CH) Piece {
      __hip_bfloat16 x[CH];
    };
    union {
      int4 raw;
      unsigned w[4];
    } q[CH];
    int held = -1;  // token of the group whose block's codes are in q
    for (int k = 0; k < 16 && t0 + k < p.num_tokens; ++k) {
      const int64_t sk = __shfl(slot, k);
      const float vs = __shfl(scale, k);
      Piece o;
      if (sk < 0) {
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) o.x[ch] = __float2bfloat16(0.f);
      } else {
        if (held < 0 || __shfl(blk, held) != sk / kBlock) {
          held = k;
          const char* tile = static_cast<const char*>(p.v_cache) + sk / kBlock * p.cache_block_stride + h * p.cache_head_stride;
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) q[ch].raw = *reinterpret_cast<const int4*>(tile + (lane * CH + ch) * kBlock);
        }
        const int ok = (int)(sk % kBlock);
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          const unsigned lo = ok & 4 ? q[ch].w[1] : q[ch].w[0], hi = ok & 4 ? q[ch].w[3] : q[ch].w[2];
          const unsigned w = (ok & 8 ? hi : lo) >> (8 * (ok & 3));
          o.x[ch] = __float2bfloat16(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * vs);
        }
      }
      *reinterpret_cast<Piece*>(static_cast<__hip_bfloat16*>(const_cast<void*>(p.value)) + (t0 + k) * p.token_stride +
                                (int64_t)h * p.head_stride + lane * CH) = o;
    }
  }
}

hipError_t launch_append_block(const BlockCacheParams& p, hipStream_t stream) {
  if (p.num_tokens == 0) return hipSuccess;
  if (p.head_dim == 64)
    hipLaunchKernelGGL(fca_append_block_kernel<64>, dim3(p.num_tokens), dim3(256), 0, stream, p);
  else if (p.head_dim == 128)
    hipLaunchKernelGGL(fca_append_block_kernel<128>, dim3(p.num_tokens), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(fca_append_block_kernel<256>, dim3(p.num_tokens), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_gather_block(const BlockCacheParams& p, hipStream_t stream) {
  if (p.num_tokens == 0) return hipSuccess;
  const int64_t tasks = ((int64_t)p.num_tokens + 15) / 16 * 2 * p.num_kv_heads;
  const unsigned grid = (unsigned)((tasks + 3) / 4);
  if (p.head_dim == 64)
    hipLaunchKernelGGL(fca_gather_block_kernel<64>, dim3(grid), dim3(256), 0, stream, p);
  else if (p.head_dim == 128)
    hipLaunchKernelGGL(fca_gather_block_kernel<128>, dim3(grid), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(fca_gather_block_kernel<256>, dim3(grid), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace fca
