// Writer and reader of the block-scaled 8-bit cache (fca_block_scales.h).
//
// Writing.  For a block b, KV head h and plane (K or V) that a call touches, with a = the largest
// finite magnitude among the call's tokens in b:
//   need   = smallest power of two s with a <= 448 s
//   old    = nothing if a token of the call has offset 0 (it begins the block), else the block's scale
//   scale' = max(old, need)
//   codes of the call's tokens = e4m3(x / scale'), nearest, ties to even, saturating; NaN stays NaN
//   where scale' > old, the codes of the other tokens become e4m3(c * old / scale')
// All tokens of a call that fall into one block are handled by the same workgroups, so the scale is
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

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef int64_t i64x2 __attribute__((ext_vector_type(2)));

__device__ inline float bf16_float(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
__device__ inline float bf16_low(unsigned w) { return __uint_as_float(w << 16); }
__device__ inline float bf16_high(unsigned w) { return __uint_as_float(w & 0xffff0000u); }

__device__ inline unsigned e4m3_code(float x) {
  // saturate (clamp, then round to nearest even); NaN is stored as the canonical 0x7f
  if (x != x) return 0x7f;
  x = fminf(fmaxf(x, -kE4m3Max), kE4m3Max);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xff;
}
__device__ inline unsigned e4m3_codes(float a, float b, float c, float d) {
  return e4m3_code(a) | e4m3_code(b) << 8 | e4m3_code(c) << 16 | e4m3_code(d) << 24;
}
// The same for numbers that are known to lie within +-448.
__device__ inline unsigned e4m3_codes_of_small(float a, float b, float c, float d) {
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
// Four codes, scaled by at most 1 and rounded again (a code that is NaN may be among them).
__device__ inline unsigned rescaled_codes(unsigned w, float ratio) {
  return e4m3_codes(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)(w >> 8), 0) * ratio,
                    __builtin_amdgcn_cvt_f32_fp8((int)(w >> 16), 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)(w >> 24), 0) * ratio);
}

// Largest magnitudes of pairs of bf16 numbers, as bit patterns: magnitudes order like integers.
__device__ inline u16x2 pair_max(u16x2 m, unsigned w) {
  const u16x2 x = __builtin_bit_cast(u16x2, w & 0x7fff7fffu);
  return u16x2{x[0] > m[0] ? x[0] : m[0], x[1] > m[1] ? x[1] : m[1]};
}
__device__ inline unsigned short finite_max(unsigned short m, unsigned w) {
  const unsigned short lo = w & 0x7fff, hi = (w >> 16) & 0x7fff;
  if (lo < 0x7f80 && lo > m) m = lo;
  if (hi < 0x7f80 && hi > m) m = hi;
  return m;
}
// The lane's largest finite magnitude in `n` dwords; `special`: an infinity or a NaN is among them.
template <int N>
__device__ inline unsigned short lane_max(const unsigned (&w)[N], bool& special) {
  u16x2 pm = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) pm = pair_max(pm, w[i]);
  unsigned short m = pm[0] > pm[1] ? pm[0] : pm[1];
  special = m >= 0x7f80;
  if (special) {
    m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = finite_max(m, w[i]);
  }
  return m;
}

// The scale of one (block, head, plane): what it was, what it becomes.
struct ScaleStep {
  float inv;     // 1 / new scale
  float ratio;   // old / new, for the codes that stay
  bool grown;    // codes that stay have to be rescaled
  bool special;  // infinities or NaNs among the tile's new values
};
__device__ inline ScaleStep step_scale(float* at, float was, unsigned lane_amax, bool lane_special, bool begins, int lane) {
  unsigned amax = lane_amax;  // (bit patterns of bf16 magnitudes: their order is that of the numbers)
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(amax, off);
    amax = o > amax ? o : amax;
  }
  // (a scale that is no positive finite number, of a block nothing has begun, counts for nothing)
  const bool has_old = !begins && was > 0.f && was < INFINITY;
  int e = scale_exp_for(bf16_float((unsigned short)amax));
  if (has_old) {
    const int eo = scale_exp_above(was);  // (a caller's own scale that is no power of two is raised to one)
    e = e > eo ? e : eo;
  }
  const float scale = __uint_as_float((unsigned)e << 23);
  ScaleStep s;
  s.inv = __uint_as_float((unsigned)(254 - e) << 23);
  s.ratio = was * s.inv;
  s.grown = has_old && scale != was;
  s.special = __ballot(lane_special) != 0;
  if (lane == 0 && scale != was) *at = scale;
  return s;
}

// A block that gets few tokens is not read unless its scale grows (then behind the reduction): its
// other codes stay where they are (512 tokens of 512 blocks: 9.2 us, 9.7 with the reads).  With more of
// them the old codes are fetched along with the rows.
constexpr int kFewTokens = 4;

// `win`: the call's token at every offset of the block, -1 = none.
template <int D>
__device__ inline void append_k_tile(const BlockCacheParams& p, const int* win, int64_t blk, int h, int lane) {
  constexpr int U = D / 64;  // 16-byte units of the tile per lane
  const int tok = lane & 15;
  const int t = win[tok];
  float* at = p.scales + (blk * p.num_kv_heads + h) * 2;
  const float was = *at;  // (every lane has it before the reduction, lane 0 writes behind it)
  char* tile = static_cast<char*>(p.k_cache) + blk * p.cache_block_stride + h * p.cache_head_stride;
  const unsigned short* row = static_cast<const unsigned short*>(p.key) + (int64_t)t * p.token_stride + (int64_t)h * p.head_stride;
  const bool few = __popcll(__ballot(t >= 0)) <= 4 * kFewTokens;
  unsigned in[U * 8];
  union Codes {
    int4 raw;
    unsigned w[4];
  } out[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = (lane >> 4) + 4 * i;
    int4 x0 = make_int4(0, 0, 0, 0), x1 = x0;
    if (t >= 0) {
      x0 = *reinterpret_cast<const int4*>(row + 16 * c);
      x1 = *reinterpret_cast<const int4*>(row + 16 * c + 8);
    } else if (!few) {
      out[i].raw = *reinterpret_cast<const int4*>(tile + (c * kBlock + tok) * 16);
    }
    in[8 * i] = x0.x, in[8 * i + 1] = x0.y, in[8 * i + 2] = x0.z, in[8 * i + 3] = x0.w;
    in[8 * i + 4] = x1.x, in[8 * i + 5] = x1.y, in[8 * i + 6] = x1.z, in[8 * i + 7] = x1.w;
  }
  bool special;
  const unsigned amax = lane_max(in, special);
  const ScaleStep s = step_scale(at, was, amax, special, win[0] >= 0, lane);
  if (t < 0) {
    if (!s.grown) return;
    if (few) {
#pragma unroll
      for (int i = 0; i < U; ++i) out[i].raw = *reinterpret_cast<const int4*>(tile + (((lane >> 4) + 4 * i) * kBlock + tok) * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int c = (lane >> 4) + 4 * i;
    if (t >= 0) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const unsigned lo = in[8 * i + 2 * d], hi = in[8 * i + 2 * d + 1];
        const float x0 = bf16_low(lo) * s.inv, x1 = bf16_high(lo) * s.inv, x2 = bf16_low(hi) * s.inv, x3 = bf16_high(hi) * s.inv;
        out[i].w[d] = s.special ? e4m3_codes(x0, x1, x2, x3) : e4m3_codes_of_small(x0, x1, x2, x3);
      }
    } else {
#pragma unroll
      for (int d = 0; d < 4; ++d) out[i].w[d] = rescaled_codes(out[i].w[d], s.ratio);
    }
    *reinterpret_cast<int4*>(tile + (c * kBlock + tok) * 16) = out[i].raw;
  }
}

// CH adjacent bf16 numbers (an element access of 2, 4 or 8 bytes) as dwords.
template <int CH>
__device__ inline void load_channels(const unsigned short* from, unsigned (&w)[(CH + 1) / 2]) {
  if constexpr (CH == 1) {
    w[0] = *from;
  } else if constexpr (CH == 2) {
    w[0] = *reinterpret_cast<const unsigned*>(from);
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(from);
    w[0] = x.x, w[1] = x.y;
  }
}

template <int D>
__device__ inline void append_v_tile(const BlockCacheParams& p, const int* win, int64_t blk, int h, int lane) {
  constexpr int CH = D / 64;  // adjacent channels per lane
  constexpr int W = (CH + 1) / 2;
  float* at = p.scales + (blk * p.num_kv_heads + h) * 2 + 1;
  const float was = *at;
  char* tile = static_cast<char*>(p.v_cache) + blk * p.cache_block_stride + h * p.cache_head_stride + lane * CH * kBlock;
  const unsigned short* rows = static_cast<const unsigned short*>(p.value) + (int64_t)h * p.head_stride + lane * CH;
  const int mine = win[lane & 15];
  const unsigned live = (unsigned)(__ballot(mine >= 0) & 0xffff);
  union Codes {
    int4 raw;
    unsigned w[4];
  } old[CH];
  const bool few = __popc(live) <= kFewTokens;
  if (live != 0xffff && !few) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) old[ch].raw = *reinterpret_cast<const int4*>(tile + ch * kBlock);
  } else {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) old[ch].raw = make_int4(0, 0, 0, 0);
  }
  unsigned in[kBlock * W];
#pragma unroll
  for (int k = 0; k < kBlock; ++k) {
    const int t = __builtin_amdgcn_readlane(mine, k);
    unsigned w[W] = {};
    if (t >= 0) load_channels<CH>(rows + (int64_t)t * p.token_stride, w);
#pragma unroll
    for (int i = 0; i < W; ++i) in[k * W + i] = w[i];
  }
  bool special;
  const unsigned amax = lane_max(in, special);
  const ScaleStep s = step_scale(at, was, amax, special, live & 1, lane);
  if (few && !s.grown) {
#pragma unroll
    for (int k = 0; k < kBlock; ++k) {
      if (!(live >> k & 1)) continue;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const unsigned w = in[k * W + ch / 2];
        tile[ch * kBlock + k] = (char)e4m3_code((ch & 1 ? bf16_high(w) : bf16_low(w)) * s.inv);
      }
    }
    return;
  }
  if (few) {
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) old[ch].raw = *reinterpret_cast<const int4*>(tile + ch * kBlock);
  }
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned w = in[(4 * d + e) * W + ch / 2];
        x[e] = (ch & 1 ? bf16_high(w) : bf16_low(w)) * s.inv;
      }
      const unsigned q = s.special ? e4m3_codes(x[0], x[1], x[2], x[3]) : e4m3_codes_of_small(x[0], x[1], x[2], x[3]);
      // bytes of the call's tokens (the same in every lane)
      const unsigned four = (live >> (4 * d)) & 15;
      const unsigned fresh = ((four & 1) | (four & 2) << 7 | (four & 4) << 14 | (four & 8) << 21) * 0xffu;
      const unsigned kept = s.grown ? rescaled_codes(old[ch].w[d], s.ratio) : old[ch].w[d];
      old[ch].w[d] = (q & fresh) | (kept & ~fresh);
    }
    *reinterpret_cast<int4*>(tile + ch * kBlock) = old[ch].raw;
  }
}

// A workgroup takes `window` successive tokens of the call and `heads` KV heads: it owns the blocks
// whose first token of the call is among them.  Which of its blocks that holds for, and which later
// tokens belong to them, it finds by looking at all slots of the call: they are few next to the rows
// (8 bytes a token against 4 D Hkv), come out of the L2, and nothing has to be known about their order.
// Cutting a long call into launches that see their own slots only would make the rule for the scales
// depend on where the cut falls.  A slot's block is looked up among the window's (at most 64) in a table
// of kTable places: one read of LDS for almost every slot, where comparing with all of them grows with
// their number (131072 tokens of 8 heads of 128: 263 us in order and 0.8 ms scattered; by comparing 332
// and 2.5 ms, cut into launches of 32768 tokens 269 and 2.1 ms).
constexpr int kMaxWindow = 64;
constexpr int kAppendThreads = 512;  // at most
constexpr int kTable = 256;          // (at most a quarter of it is taken, so every search ends)
__device__ inline int place_of(int blk) { return (int)((unsigned)blk * 0x9E3779B1u >> 24); }
template <int D>
__global__ __launch_bounds__(kAppendThreads) void fca_append_block_kernel(BlockCacheParams p, int window, int heads, int head_groups) {
  __shared__ int cand[kMaxWindow];         // blocks of the window's tokens, each once
  __shared__ int win[kMaxWindow][kBlock];  // the call's last token at every offset of theirs, -1 = none
  __shared__ int foreign[kMaxWindow];      // the block has a token in front of the window
  __shared__ int num_cand;
  __shared__ int table[kTable];            // a candidate's number + 1 at the first free place from its block's on, 0 = none
  const int tid = threadIdx.x, threads = blockDim.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int w = blockIdx.x / head_groups, h0 = (blockIdx.x - w * head_groups) * heads;
  const int t0 = w * window;
  const int64_t end = p.num_blocks * kBlock;
  if (wave == 0) {
    int blk = -1;
    if (lane < window && t0 + lane < p.num_tokens) {
      const int64_t slot = p.slot_mapping[t0 + lane];
      if (slot >= 0 && slot < end) blk = (int)(slot / kBlock);
    }
    bool leads = blk >= 0;
    for (int j = 0; j < window - 1; ++j) {
      const int other = __builtin_amdgcn_readlane(blk, j);
      if (j < lane && other == blk) leads = false;
    }
    const unsigned long long all = __ballot(leads);
    for (int j = lane; j < kTable; j += 64) table[j] = 0;
    __builtin_amdgcn_wave_barrier();
    if (leads) {
      const int c = __popcll(all & ((1ull << lane) - 1));
      cand[c] = blk;
      int at = place_of(blk);
      while (atomicCAS(&table[at], 0, c + 1) != 0) at = (at + 1) % kTable;
    }
    if (lane == 0) num_cand = __popcll(all);
  }
  for (int j = tid; j < window * kBlock; j += threads) (&win[0][0])[j] = -1;
  if (tid < kMaxWindow) foreign[tid] = 0;
  __syncthreads();
  const int n = num_cand;
  if (n == 0) return;
  // (pairs of adjacent slots; kScan loads of a thread in flight together.  Workgroups begin at different
  // places, or all would ask the same channel of the cache for the same line at the same time.)
  constexpr int kScan = 2;
  const int trip = 2 * kScan * threads;
  const int trips = (p.num_tokens + trip - 1) / trip;
  for (int i = 0; i < trips; ++i) {
    const int base = (int)((i + blockIdx.x) % trips) * trip;
    i64x2 slots[kScan];
#pragma unroll
    for (int k = 0; k < kScan; ++k) {
      const int t = base + 2 * (k * threads + tid);
      slots[k] = i64x2{-1, -1};
      if (t + 1 < p.num_tokens)
        __builtin_memcpy(&slots[k], p.slot_mapping + t, 16);
      else if (t < p.num_tokens)
        slots[k][0] = p.slot_mapping[t];
    }
#pragma unroll
    for (int k = 0; k < 2 * kScan; ++k) {
      const int t = base + 2 * ((k >> 1) * threads + tid) + (k & 1);
      const int64_t slot = slots[k >> 1][k & 1];
      const uint64_t blk = (uint64_t)slot / kBlock;  // (a negative slot is far away)
      for (int at = place_of((int)blk);; at = (at + 1) % kTable) {
        const int c = table[at] - 1;
        if (c < 0) break;
        if ((uint64_t)cand[c] != blk) continue;
        if (t < t0) foreign[c] = 1;
        else atomicMax(&win[c][slot & (kBlock - 1)], t);
        break;
      }
    }
  }
  __syncthreads();
  const int tasks = n * heads * 2;
  for (int j = wave; j < tasks; j += threads / 64) {
    const int c = j / (2 * heads), rest = j - c * 2 * heads, h = h0 + (rest >> 1);
    if (foreign[c] || h >= p.num_kv_heads) continue;
    if (rest & 1)
      append_v_tile<D>(p, win[c], cand[c], h, lane);
    else
      append_k_tile<D>(p, win[c], cand[c], h, lane);
  }
}

// Reading back: row t = codes at slot_mapping[t] times their block's scales, rounded to bf16 (exact
// for the writer's scales, short of bf16's own range); a negative slot, or one past the cache, gives
// zeros.  A wave takes 16 tokens of one head and plane.  Of K a lane converts 16-byte units, as in
// the writer.  Of V a lane holds whole channels of one block at a time and writes every token of the
// group that lies in the block, offset by offset, so that a code's place in its register is known at
// compile time and a row leaves as one contiguous store of the wave; a run of consecutive tokens
// touches at most two blocks, both fetched in advance.  8 x 4093 tokens of 8 heads of 128 take 42 us, the
// time a copy of the bytes takes; 257 tokens of 2 heads of 64 3.9 us, a launch and three round trips.
template <int D>
__global__ __launch_bounds__(256) void fca_gather_block_kernel(BlockCacheParams p) {
  constexpr int CH = D / 64;  // adjacent channels per lane (V)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  const int64_t group = task / (2 * p.num_kv_heads);
  const int j = (int)(task - group * 2 * p.num_kv_heads), h = j >> 1;
  const int64_t t0 = group * kBlock;
  if (t0 >= p.num_tokens) return;
  const int64_t t = t0 + (lane & 15);
  const int64_t slot = t < p.num_tokens ? p.slot_mapping[t] : -1;
  const bool live = slot >= 0 && slot < p.num_blocks * kBlock;
  const int blk = live ? (int)(slot / kBlock) : -1, off = live ? (int)(slot % kBlock) : 0;
  const float scale = live ? p.scales[((int64_t)blk * p.num_kv_heads + h) * 2 + (j & 1)] : 0.f;
  if ((j & 1) == 0) {
    constexpr int U = D / 64;
    if (t >= p.num_tokens) return;
    const char* tile = static_cast<const char*>(p.k_cache) + (int64_t)max(blk, 0) * p.cache_block_stride + h * p.cache_head_stride;
    __hip_bfloat16* row = static_cast<__hip_bfloat16*>(const_cast<void*>(p.key)) + t * p.token_stride + (int64_t)h * p.head_stride;
    int4 q[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      q[i] = live ? *reinterpret_cast<const int4*>(tile + (((lane >> 4) + 4 * i) * kBlock + off) * 16) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int c = (lane >> 4) + 4 * i;
      const int w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
      union {
        int4 raw[2];
        __hip_bfloat16 x[16];
      } o;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[d], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[d], true);
        o.x[4 * d] = __float2bfloat16(a[0] * scale), o.x[4 * d + 1] = __float2bfloat16(a[1] * scale);
        o.x[4 * d + 2] = __float2bfloat16(b[0] * scale), o.x[4 * d + 3] = __float2bfloat16(b[1] * scale);
      }
      reinterpret_cast<int4*>(row + 16 * c)[0] = o.raw[0];
      reinterpret_cast<int4*>(row + 16 * c)[1] = o.raw[1];
    }
    return;
  }
  struct alignas(2 * CH) Piece {
    __hip_bfloat16 x[CH];
  };
  struct Codes {
    int w[CH][4];
  };
  __hip_bfloat16* rows = static_cast<__hip_bfloat16*>(const_cast<void*>(p.value)) + t0 * p.token_stride + (int64_t)h * p.head_stride + lane * CH;
  auto load = [&](int b) {
    const char* tile = static_cast<const char*>(p.v_cache) + (int64_t)max(b, 0) * p.cache_block_stride + h * p.cache_head_stride;
    Codes c;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int4 x = *reinterpret_cast<const int4*>(tile + (lane * CH + ch) * kBlock);
      c.w[ch][0] = x.x, c.w[ch][1] = x.y, c.w[ch][2] = x.z, c.w[ch][3] = x.w;
    }
    return c;
  };
  const int tokens = (int)min((int64_t)kBlock, (int64_t)p.num_tokens - t0);
  const bool is_token = lane < tokens;
  const int first = __builtin_amdgcn_readlane(blk, 0), last = __builtin_amdgcn_readlane(blk, tokens - 1);
  const Codes ca = load(first), cb = load(last);  // (block 0 where there is none: its codes are not used)
  unsigned todo = (unsigned)__ballot(is_token && blk >= 0);
  const unsigned padding = (unsigned)__ballot(is_token && blk < 0);
  // the tokens still to do that lie in block b, one per offset (of two with one slot the second waits)
  auto write = [&](const Codes& c, int b) {
    const bool here = ((todo >> (lane & 31)) & 1) && lane < kBlock && blk == b;
    const float vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale), __builtin_ctzll(__ballot(here))));
#pragma unroll
    for (int o = 0; o < kBlock; ++o) {
      const unsigned at = (unsigned)__ballot(here && off == o);
      if (at == 0) continue;
      const int k = __builtin_ctz(at);
      todo &= ~(1u << k);
      Piece x;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const unsigned w = (unsigned)c.w[ch][o >> 2] >> (8 * (o & 3));
        x.x[ch] = __float2bfloat16(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * vs);
      }
      *reinterpret_cast<Piece*>(rows + (int64_t)k * p.token_stride) = x;
    }
  };
  if (first >= 0) write(ca, first);
  if (todo != 0 && last >= 0 && last != first) write(cb, last);
  while (todo != 0) {
    const int b = __builtin_amdgcn_readlane(blk, __builtin_ctz(todo));
    write(load(b), b);
  }
  for (unsigned left = padding; left != 0; left &= left - 1) {
    Piece zero;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) zero.x[ch] = __float2bfloat16(0.f);
    *reinterpret_cast<Piece*>(rows + (int64_t)__builtin_ctz(left) * p.token_stride) = zero;
  }
}

hipError_t launch_append_block(const BlockCacheParams& p, hipStream_t stream) {
  if (p.num_tokens == 0) return hipSuccess;
  // Windows: at most 512 of them up to their largest size; KV heads: as many groups as bring the launch
  // to 512 workgroups; waves: one for each two tiles of a workgroup, 4 to 8.  Few large workgroups
  // look at all the slots: 8191 tokens of 8 heads take 16.5 us (comparing with all blocks of a window it was
  // 17.5, and with 1024 workgroups of 4 waves 21, with twice as many windows 26); 8 tokens take 4.7 (an
  // empty launch: 2.5), 512 tokens of 512 blocks 9.4.
  int window = 1;
  while (window < kMaxWindow && (p.num_tokens + window - 1) / window > 512) window *= 2;
  const int windows = (p.num_tokens + window - 1) / window;
  int groups = (512 + windows - 1) / windows;
  if (groups > p.num_kv_heads) groups = p.num_kv_heads;
  const int heads = (p.num_kv_heads + groups - 1) / groups;
  groups = (p.num_kv_heads + heads - 1) / heads;
  const dim3 grid(windows * groups);
  int threads = 64 * heads * (window > 1 ? 2 : 1);
  threads = threads < 256 ? 256 : threads > kAppendThreads ? kAppendThreads : threads;
  if (p.head_dim == 64)
    hipLaunchKernelGGL(fca_append_block_kernel<64>, grid, dim3(threads), 0, stream, p, window, heads, groups);
  else if (p.head_dim == 128)
    hipLaunchKernelGGL(fca_append_block_kernel<128>, grid, dim3(threads), 0, stream, p, window, heads, groups);
  else
    hipLaunchKernelGGL(fca_append_block_kernel<256>, grid, dim3(threads), 0, stream, p, window, heads, groups);
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
