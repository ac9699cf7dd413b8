// Forest cascade attention over the block-scaled 8-bit cache (fca_block_scales.h): the work items,
// tile orders, matrix products and partial rows of the per-head fp8 kernels (fca_attend.hip), with
// a K scale and a V scale per block of 16 tokens.
//
//   S[t, row] = softmax_scale * s_k[block of t] * sum_d c_k[t, d] q[row, d]
//   O[d, row] = sum_t c_v[d, t] * (s_v[block of t] * P[t, row])
//
// A 32-token tile covers two blocks, and the accumulator registers 0-7 and 8-15 of a lane hold the
// tokens of the first and the second: the K scale is one of two wave-uniform factors of the
// exponent's fused multiply-add, the V scale one multiplication of a probability before it is
// rounded to bf16 for the value product (that rounding is relative, so the scale costs no
// precision).  The codes go through the matrix cores as bf16, which holds every e4m3 value exactly.
#include <hip/hip_ext.h>

#include <type_traits>

#include "fca_attend_common.h"
#include "fca_block_scales.h"

namespace fca {

// A row whose scores held a NaN has a sum that is none.  The merge drops a partial without a
// log-sum-exp as an empty one; this tag in the row's scale, which points to no second partial, makes
// it give NaN for the row and its log-sum-exp instead.
constexpr int kNanTag = 1;

// 0xff in every byte of a dword of codes that holds a NaN (0x7f or 0xff).
__device__ inline unsigned nan_bytes(unsigned w) {
  const unsigned x = (w & 0x7f7f7f7fu) + 0x01010101u;  // bit 7 of a byte: its magnitude was 0x7f
  return ((x & 0x80808080u) >> 7) * 0xffu;
}
template <class VT>
__device__ inline bool holds_nan(const VT& vt) {
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < VT::NV; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) any |= nan_bytes((unsigned)vt.v[0][i][j]) | nan_bytes((unsigned)vt.v[1][i][j]);
  return any != 0;
}

template <int D, bool STREAM, int NRT>
__global__ __launch_bounds__(kThreads, 1) void fca_attend_block_kernel(AttendParams p) {
  constexpr int KS = D / 16;   // MFMA steps of the score product
  constexpr int NDB = D / 32;  // 32-channel blocks of the output
  using KT = KTile<D, true>;
  using VT = VTile<D, true>;

  const int32_t* hdr = p.meta + p.off_header;
  const int total = hdr[H_ITEMS], shared = hdr[H_SHARED_ITEMS];
  const int first = p.select == 2 ? shared : 0;
  const int last_item = p.select == 1 ? shared : total;
  const int ntickets = (last_item - first) * p.num_kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m = lane & 31, h = lane >> 5;
  const int G = p.group, Hkv = p.num_kv_heads;
  const int32_t* meta = p.meta;

  int row_member[NRT], row_head[NRT];
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    row_member[rt] = (rt * 32 + m) / G;
    row_head[rt] = (rt * 32 + m) - row_member[rt] * G;
  }
  const int tok_of_m = (m & 3) | ((m & 4) << 1) | ((m & 8) >> 1);
  const int k_lane_off = h * 256 + tok_of_m * 16;
  const int v_lane_off = (h * 32 + m) * 16;
  __shared__ __attribute__((aligned(16))) char strips[kWaves][NRT * 32 * strip_row_bytes<D>()];
  char* strip = strips[wave];
  const float2* scales = reinterpret_cast<const float2*>(p.k_scale);

  const int nwaves = (int)gridDim.x * kWaves;
  for (int ticket = (int)blockIdx.x * kWaves + wave; ticket < ntickets; ticket += nwaves) {
    const int item = ticket / Hkv, kvh = ticket - item * Hkv;
    const int4* rec = reinterpret_cast<const int4*>(meta + p.off_items + (int64_t)(first + item) * kItemInts);
    const int4 r0 = rec[0], r1 = rec[1];
    const int tok_len = __builtin_amdgcn_readfirstlane(r0.z);
    const int mcnt = __builtin_amdgcn_readfirstlane(r1.x);
    const int ord = __builtin_amdgcn_readfirstlane(r1.y);
    const int sees = __builtin_amdgcn_readfirstlane(r1.w);
    const int rows = mcnt * G;
    const int nblk = (tok_len + kBlock - 1) / kBlock;
    const int ntiles = (tok_len + kTile - 1) / kTile;
    const int nfull = (tok_len - (sees > 0 ? 1 : 0)) / kTile;
    // lane b holds the id and the scales of block b of the chunk
    const int my_blk = p.block_table[(int64_t)r0.x * p.bt_stride + r0.y + min(lane, nblk - 1)];
    const float2 my_scale = scales[(int64_t)my_blk * Hkv + kvh];
    const float my_ks = my_scale.x * (p.scale * kLog2e);
    int64_t prow[NRT];
    bf16x8 qreg[NRT][KS];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      const bool live = row_member[rt] < mcnt;
      const int seq = meta[p.off_members + r0.w + (live ? row_member[rt] : 0)];
      prow[rt] = live ? ((int64_t)seq * p.max_partials + ord) * p.num_q_heads + kvh * G + row_head[rt] : -1;
      const __bf16* qp = reinterpret_cast<const __bf16*>(p.q) + (int64_t)seq * p.q_seq_stride +
                         (int64_t)(kvh * G + row_head[rt]) * p.q_head_stride;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
        if (!live) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        qreg[rt][i] = v;
      }
    }
    f32x16 acc[NRT][NDB];
    float mrow[NRT], lrow[NRT];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      mrow[rt] = -INFINITY, lrow[rt] = 0.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[rt][db][r] = 0.f;
    }

    // Value product of a tile.  NANS: NaN values are taken out of the product, and the rows that see
    // their tokens are found by a product of their own: (1 where the value is NaN) x (1 where the row
    // sees the token) counts them per row and channel.
    auto weighted_values = [&](const VT& vt, int tok0, const bf16x8 (&pb)[NRT][2], auto ragged, auto nans) {
      constexpr bool RAGGED = decltype(ragged)::value, NANS = decltype(nans)::value;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        // tokens this lane feeds for this block: 8h .. 8h+7; on the ragged tile the ones past the end
        // are zeroed, whatever the cache holds there
        const int nv = tok_len - (tok0 + 16 * blk + 8 * h);
        bf16x8 vis[NRT];
        if constexpr (NANS) {
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
            for (int k = 0; k < 8; ++k) vis[rt][k] = (__bf16)(tok0 + 16 * blk + 8 * h + k < sees + row_member[rt] ? 1.f : 0.f);
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const i32x4 raw = vt.v[blk][db >> 1];
          const auto s0 = __builtin_amdgcn_permlane32_swap((unsigned)raw[0], (unsigned)raw[2], false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap((unsigned)raw[1], (unsigned)raw[3], false, false);
          i32x2 w = {(int)s0[db & 1], (int)s1[db & 1]};
          if constexpr (RAGGED) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              unsigned keep = 0;
#pragma unroll
              for (int b = 0; b < 4; ++b)
                if (4 * j + b < nv) keep |= 0xffu << (8 * b);
              w[j] &= keep;
            }
          }
          if constexpr (NANS) {
            __builtin_amdgcn_sched_barrier(0);
            const int n0 = (int)nan_bytes((unsigned)w[0]), n1 = (int)nan_bytes((unsigned)w[1]);
            w[0] &= ~n0, w[1] &= ~n1;
            const bf16x8 is_nan = fp8x8_to_bf16(n0 & 0x38383838, n1 & 0x38383838);  // 0x38 is 1.0
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
              f32x16 cnt;
#pragma unroll
              for (int r = 0; r < 16; ++r) cnt[r] = 0.f;
              cnt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(is_nan, vis[rt], cnt, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 16; ++r)
                if (cnt[r] > 0.f) acc[rt][db][r] = __builtin_nanf("");
            }
          }
          const bf16x8 a = fp8x8_to_bf16(w[0], w[1]);
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt)
            acc[rt][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb[rt][blk], acc[rt][db], 0, 0, 0);
        }
      }
    };

    auto compute_tile = [&](const KT& kt, const VT& vt, int ti, auto ragged) {
      constexpr bool RAGGED = decltype(ragged)::value;
      const int tok0 = ti * kTile;
      float ks[2], vs[2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const int b = min(2 * ti + blk, nblk - 1);
        ks[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_ks), b));
        vs[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_scale.y), b));
      }
      bf16x8 pb[NRT][2];
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt) {
        f32x16 sr;
#pragma unroll
        for (int r = 0; r < 16; ++r) sr[r] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const i32x4 w = kt.k[i >> 1];
          const bf16x8 a = (i & 1) ? fp8x8_to_bf16(w[2], w[3]) : fp8x8_to_bf16(w[0], w[1]);
          sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qreg[rt][i], sr, 0, 0, 0);
        }
        const int row_lim = RAGGED && sees > 0 ? min(tok_len, sees + row_member[rt]) : tok_len;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (RAGGED && tok0 + 16 * (r >> 3) + 8 * h + (r & 7) >= row_lim) sr[r] = -INFINITY;
          mx[r >> 3] = fmaxf(mx[r >> 3], sr[r]);
        }
        float mtile = fmaxf(mx[0] * ks[0], mx[1] * ks[1]);
        mtile = fmaxf(mtile, __shfl_xor(mtile, 32));
        if (ti == 0) mrow[rt] = mtile;
        if (__builtin_amdgcn_readfirstlane(__any(mtile > mrow[rt] + kRescaleSlack))) {
          const float mnew = fmaxf(mrow[rt], mtile);
          const float alpha = fast_exp2(mrow[rt] - mnew);
          lrow[rt] *= alpha;
          mrow[rt] = mnew;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[rt][db][r] *= alpha;
        }
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float e = fast_exp2(__builtin_fmaf(sr[r], ks[r >> 3], -mrow[rt]));
          // (a masked score times a scale of zero is no number)
          if (RAGGED && sr[r] == -INFINITY) e = 0.f;
          sum += e;
          pb[rt][r >> 3][r & 7] = (__bf16)(e * vs[r >> 3]);
        }
        lrow[rt] += sum;
      }
      // Rows of a query run see different numbers of tokens of their last tile.  A NaN among its
      // values must not reach the rows that do not see its token (0 * NaN), so such a tile takes a
      // path of its own.
      if constexpr (RAGGED) {
        if (sees > 0 && __builtin_amdgcn_readfirstlane(__any(holds_nan(vt)))) {
          weighted_values(vt, tok0, pb, ragged, std::true_type{});
          return;
        }
      }
      weighted_values(vt, tok0, pb, ragged, std::false_type{});
    };

    for (int ti = 0; ti < ntiles; ++ti) {
      const int b0 = __builtin_amdgcn_readlane(my_blk, 2 * ti);
      const int b1 = __builtin_amdgcn_readlane(my_blk, min(2 * ti + 1, nblk - 1));
      KT kt;
      VT vt;
      const char* kp = p.k_cache + (int64_t)kvh * p.kv_head_bytes + (int64_t)((m & 16) ? b1 : b0) * p.kv_block_bytes + k_lane_off;
#pragma unroll
      for (int i = 0; i < KT::NK; ++i) kt.k[i] = load16<STREAM>(kp + i * 512);
      const char* vbase = p.v_cache + (int64_t)kvh * p.kv_head_bytes + v_lane_off;
#pragma unroll
      for (int i = 0; i < VT::NV; ++i) {
        vt.v[0][i] = load16<STREAM>(vbase + (int64_t)b0 * p.kv_block_bytes + i * 1024);
        vt.v[1][i] = load16<STREAM>(vbase + (int64_t)b1 * p.kv_block_bytes + i * 1024);
      }
      if (ti < nfull)
        compute_tile(kt, vt, ti, std::false_type{});
      else
        compute_tile(kt, vt, ti, std::true_type{});
    }
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      const float l = lrow[rt] + __shfl_xor(lrow[rt], 32);
      stage_partial_row<D, STREAM>(strip, rt * 32 + m, h, acc[rt], 1.f / l, prow[rt], (mrow[rt] + fast_log2(l)) * kLn2, p.partial_lse,
                                   l != l ? kNanTag : 0);
    }
    __builtin_amdgcn_wave_barrier();
    store_partial_rows<D, STREAM>(strip, rows, lane, p.partial_out);
    __builtin_amdgcn_wave_barrier();
  }
}

hipError_t launch_attend_block(const AttendParams& p, const fca_plan& plan, int max_workgroups, hipStream_t stream) {
  const MetaLayout L = make_layout(plan);
  const int64_t max_tickets = L.max_items * plan.num_kv_heads;
  int grid = 256;
  if (max_workgroups > 0 && max_workgroups < grid) grid = max_workgroups;
  if ((int64_t)grid * kWaves > max_tickets) grid = (int)((max_tickets + kWaves - 1) / kWaves);
  const bool stream_kv = plan.max_levels > 0 && !p.kv_reread;
  hipEvent_t ev_start, ev_stop;
  take_attend_timing(&ev_start, &ev_stop);
#define FCA_LAUNCH(D_, S_, N_) \
  if (ev_start) hipExtLaunchKernelGGL((fca_attend_block_kernel<D_, S_, N_>), dim3(grid), dim3(kThreads), 0, stream, ev_start, ev_stop, 0, p); \
  else hipLaunchKernelGGL((fca_attend_block_kernel<D_, S_, N_>), dim3(grid), dim3(kThreads), 0, stream, p)
#define FCA_PICK(D_, N_) \
  if (stream_kv) { FCA_LAUNCH(D_, true, N_); } else { FCA_LAUNCH(D_, false, N_); }
  if (plan.head_dim == 256) {
    FCA_PICK(256, 1);
  } else if (plan.head_dim == 128) {
    if (plan.rows_per_item == 64) { FCA_PICK(128, 2); } else { FCA_PICK(128, 1); }
  } else {
    if (plan.rows_per_item == 64) { FCA_PICK(64, 2); } else { FCA_PICK(64, 1); }
  }
#undef FCA_PICK
#undef FCA_LAUNCH
  return hipGetLastError();
}

}  // namespace fca
