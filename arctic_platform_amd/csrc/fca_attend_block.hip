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
// The value the lane 32 away holds, without a trip through LDS.
__device__ inline float other_half(float x) {
  const unsigned u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
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

// Workgroups per CU (a wave's registers are 512 / this) and whether the next item's query rows are
// held in registers of their own an item ahead.
template <int D, int NRT>
struct BlockTuning {
  static constexpr int kWorkgroups = D == 64 ? 2 : 1;
  static constexpr bool kEarlyQ = D <= 128 && NRT == 1;
  static constexpr bool kCoop = kWorkgroups == 1 && NRT == 1;
};

template <int D, bool STREAM, int NRT>
__global__ __launch_bounds__(kThreads, (BlockTuning<D, NRT>::kWorkgroups)) void fca_attend_block_kernel(AttendParams p) {
  using Tune = BlockTuning<D, NRT>;
  constexpr int KS = D / 16;   // MFMA steps of the score product
  constexpr int NDB = D / 32;  // 32-channel blocks of the output
  using KT = KTile<D, true>;
  using VT = VTile<D, true>;

  int32_t* hdr = p.meta + p.off_header;
  const int total = hdr[H_ITEMS], shared = hdr[H_SHARED_ITEMS];
  const int first = p.select == 2 ? shared : 0;
  const int last_item = p.select == 1 ? shared : total;
  const int ntickets = (last_item - first) * p.num_kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m = lane & 31, h = lane >> 5;
  const int G = p.group, Hkv = p.num_kv_heads;
  const int32_t* meta = p.meta;
  const int nwaves = (int)gridDim.x * kWaves;
  const int my_wave = (int)blockIdx.x * kWaves + wave;
  if (my_wave >= ntickets) return;

  // row rt * 32 + m of the stacked query tile is (member row / G, head row % G)
  int row_member[NRT], row_head[NRT];
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    row_member[rt] = (rt * 32 + m) / G;
    row_head[rt] = (rt * 32 + m) - row_member[rt] * G;
  }
  // MFMA row m carries the token whose index has bits 2 and 3 of m swapped: the score
  // accumulator then holds, per lane half, tokens 8h..8h+7 of each block in register order.
  const int tok_of_m = (m & 3) | ((m & 4) << 1) | ((m & 8) >> 1);
  const int k_lane_off = h * 256 + tok_of_m * 16;
  const int v_lane_off = (h * 32 + m) * 16;  // channel 32 * (2 * pair + h) + m, all 16 tokens
  // wave-private strip of LDS for the output rows
  __shared__ __attribute__((aligned(16))) char strips[kWaves][NRT * 32 * strip_row_bytes<D>()];
  char* strip = strips[wave];
  const float2* scales = reinterpret_cast<const float2*>(p.k_scale);

  // Dealing the work, as in fca_attend32.hip: the largest tickets go one to a pair of waves on
  // different XCDs, which take them last and from both ends; the rest is dealt back and forth over
  // the size-ordered list, and its last full round and remainder are drawn from a counter.
  const int half_grid = (int)gridDim.x >> 1;
  const bool coop_back = (int)blockIdx.x >= half_grid;
  const int pair_id = (coop_back ? (((int)blockIdx.x ^ 3) - half_grid) : (int)blockIdx.x) * kWaves + wave;
  const bool coop_on = Tune::kCoop && p.coop_ctr != nullptr && (gridDim.x & 7) == 0 && nwaves / 2 * NRT <= p.coop_pairs &&
                       ntickets >= nwaves / 2 + 3 * nwaves;
  const int coop = coop_on ? nwaves / 2 : 0;
  const int nmain = ntickets - coop;
  const int static_tickets = nmain < 5 * nwaves ? nmain : (nmain / nwaves - 1) * nwaves;
  const int dynamic_draws = nmain - static_tickets + nwaves;
  bool drawing = static_tickets < nmain;
  bool coop_pending = coop_on;
  // A zero the compiler cannot see through; it makes an address look lane-dependent, which keeps
  // what is loaded there out of scalar registers: the move would wait for every load in flight.
  int opaque_zero;
  asm volatile("v_mov_b32 %0, 0" : "=v"(opaque_zero));
  int tv_drawn = 0;
  auto issue_ticket = [&](int r) {
    if (r * nwaves >= static_tickets && drawing && lane == 0) tv_drawn = atomicAdd(&hdr[H_TICKET + opaque_zero], 1);
  };
  auto after_main = [&]() -> int {
    if (!coop_pending) return ntickets;
    coop_pending = false;
    return pair_id;
  };
  auto resolve_ticket = [&](int r) -> int {
    if (r * nwaves < static_tickets) {
      const int t = r * nwaves + ((r & 1) ? nwaves - 1 - my_wave : my_wave);
      return t < nmain ? coop + t : after_main();
    }
    if (!drawing) return after_main();
    const int drawn = __builtin_amdgcn_readfirstlane(tv_drawn);
    if (drawn == dynamic_draws - 1 && lane == 0) hdr[H_TICKET] = 0;  // nobody draws after this one
    const int t = static_tickets + drawn;
    if (t >= nmain) {
      drawing = false;
      return after_main();
    }
    return coop + t;
  };
  auto load_record = [&](int t, int4& r0, int4& r1, int& kvh) {
    const int tc = min(t, ntickets - 1);
    const int it = tc / Hkv;
    kvh = tc - it * Hkv;
    const int4* rec =
        reinterpret_cast<const int4*>(meta + p.off_items + (int64_t)(first + it) * kItemInts + opaque_zero);
    r0 = rec[0];  // rep, blk_start, tok_len, member_off
    r1 = rec[1];  // member_cnt, ord, node, tokens the first member sees (causal last chunk) or 0
  };
  // Per-lane data that hangs off a record: one block id of the chunk per lane (a chunk has at most
  // 64 blocks) and the member sequences of this lane's query rows.
  auto load_lane_meta = [&](const int4& r0, const int4& r1, int& my_blk, int (&seq)[NRT]) {
    const int nblk = (r0.z + kBlock - 1) / kBlock;
    my_blk = p.block_table[(int64_t)r0.x * p.bt_stride + r0.y + min(lane, nblk - 1)];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) seq[rt] = meta[p.off_members + r0.w + (row_member[rt] < r1.x ? row_member[rt] : 0)];
  };
  // ... and off the block ids: the scales of the lane's block
  auto load_scales = [&](int my_blk, int kvh) -> float2 { return scales[(int64_t)my_blk * Hkv + kvh]; };
  auto load_q = [&](bf16x8 (&q)[NRT][KS], const int (&seq)[NRT], int mcnt, int kvh) {
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      const bool live = row_member[rt] < mcnt;
      const __bf16* qp = reinterpret_cast<const __bf16*>(p.q) + (int64_t)seq[rt] * p.q_seq_stride +
                         (int64_t)(kvh * G + row_head[rt]) * p.q_head_stride;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        // the K tile hands a lane 16 channels of one token: two steps
        bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
        if (!live) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        q[rt][i] = v;
      }
    }
  };
  // (the fences keep the loads in front of the next tile's arithmetic, which starts with a wait)
  auto load_tile = [&](KT& kt, VT& vt, int my_blk, int nblk, int kvh, int ti) {
    __builtin_amdgcn_sched_barrier(0);
    const int b0 = __builtin_amdgcn_readlane(my_blk, 2 * ti);
    const int b1 = __builtin_amdgcn_readlane(my_blk, min(2 * ti + 1, nblk - 1));
    const char* kp = p.k_cache + (int64_t)kvh * p.kv_head_bytes + (int64_t)((m & 16) ? b1 : b0) * p.kv_block_bytes + k_lane_off;
#pragma unroll
    for (int i = 0; i < KT::NK; ++i) kt.k[i] = load16<STREAM>(kp + i * 512);
    const char* vbase = p.v_cache + (int64_t)kvh * p.kv_head_bytes + v_lane_off;
    const char* vp0 = vbase + (int64_t)b0 * p.kv_block_bytes;
    const char* vp1 = vbase + (int64_t)b1 * p.kv_block_bytes;
#pragma unroll
    for (int i = 0; i < VT::NV; ++i) {
      vt.v[0][i] = load16<STREAM>(vp0 + i * 1024);
      vt.v[1][i] = load16<STREAM>(vp1 + i * 1024);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- set-up: the first three items of this wave; their tickets are static
  int4 r0, r1, a0, a1, b0, b1;  // records of the current item and the two after it
  int kvh, akvh, bkvh;
  int my_blk, a_blk, seq[NRT], a_seq[NRT];
  int t_cur = resolve_ticket(0);  // rounds 0 to 3 are static, or the whole list is
  int ta = resolve_ticket(1);
  int tb = resolve_ticket(2);
  load_record(t_cur, r0, r1, kvh);
  load_record(ta, a0, a1, akvh);
  load_record(tb, b0, b1, bkvh);
  load_lane_meta(r0, r1, my_blk, seq);
  load_lane_meta(a0, a1, a_blk, a_seq);
  bf16x8 qreg[NRT][KS], nq[Tune::kEarlyQ ? NRT : 1][KS];
  load_q(qreg, seq, r1.x, kvh);
  float2 my_scale = load_scales(my_blk, kvh), next_scale = my_scale;
  KT kb0, kb1;
  VT vb0, vb1;
  {
    const int len = __builtin_amdgcn_readfirstlane(r0.z);
    const int nb = (len + kBlock - 1) / kBlock;
    load_tile(kb0, vb0, my_blk, nb, kvh, 0);
    load_tile(kb1, vb1, my_blk, nb, kvh, min(1, (len + kTile - 1) / kTile - 1));
  }

  // ---- state of the item being attended
  struct Item {
    int tok_len;  // KV tokens of the chunk
    int nblk;
    // Last chunk of a query-run tile: member i sees the first `sees + i` tokens of the chunk
    // (its own token and what is before it); all members end inside the last tile.
    int sees;
    f32x16 acc[NRT][NDB];
    float mrow[NRT], lrow[NRT];  // reference maximum (scaled, log2 domain) and running sum
    float ks;                    // K scale of the lane's block, times softmax scale and log2(e)
  };
  auto begin_item = [&](Item& it) {
    it.tok_len = __builtin_amdgcn_readfirstlane(r0.z);
    it.nblk = (it.tok_len + kBlock - 1) / kBlock;
    it.sees = __builtin_amdgcn_readfirstlane(r1.w);
    it.ks = my_scale.x * (p.scale * kLog2e);
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      it.mrow[rt] = -INFINITY, it.lrow[rt] = 0.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) it.acc[rt][db][r] = 0.f;
    }
  };

  // Operand registers of the value product: rows of channel blocks 2 * pair and 2 * pair + 1 sit in the
  // lower and upper lane halves; the swap hands every lane its tokens 8h..8h+7 of channel block db.
  // RAGGED: tokens past the end of the chunk are zeroed, whatever the cache holds there.
  auto value_codes = [&](const Item& it, const VT& vt, int tok0, int blk, int db, auto ragged) -> i32x2 {
    const i32x4 raw = vt.v[blk][db >> 1];
    const auto s0 = __builtin_amdgcn_permlane32_swap((unsigned)raw[0], (unsigned)raw[2], false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap((unsigned)raw[1], (unsigned)raw[3], false, false);
    i32x2 w = {(int)s0[db & 1], (int)s1[db & 1]};
    if constexpr (decltype(ragged)::value) {
      const int nv = it.tok_len - (tok0 + 16 * blk + 8 * h);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        unsigned keep = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (4 * j + b < nv) keep |= 0xffu << (8 * b);
        w[j] &= keep;
      }
    }
    return w;
  };
  auto weighted_values = [&](Item& it, const VT& vt, int tok0, const bf16x8 (&pb)[NRT][2], auto row_tiles, auto ragged) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        i32x2 w = value_codes(it, vt, tok0, blk, db, ragged);
        if constexpr (decltype(ragged)::value) {
          const int run = it.sees > 0 ? -1 : 0;  // (seen_nans puts them where they belong)
          w[0] &= ~((int)nan_bytes((unsigned)w[0]) & run);
          w[1] &= ~((int)nan_bytes((unsigned)w[1]) & run);
        }
        const bf16x8 a = fp8x8_to_bf16(w[0], w[1]);
#pragma unroll
        for (int rt = 0; rt < decltype(row_tiles)::value; ++rt)
          it.acc[rt][db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb[rt][blk], it.acc[rt][db], 0, 0, 0);
      }
  };
  // Rows of a query run see different numbers of tokens of their last tile, and a NaN among its values
  // must not reach the rows that do not see its token (0 * NaN).  So there the NaNs are left out of the
  // value product; where a row does see one, the product of (huge where the value is NaN) and (huge
  // where the row sees the token) overflows, and infinity * 0 makes the row's sum of that channel NaN.
  auto seen_nans = [&](Item& it, const VT& vt, int tok0) {
    constexpr float kHuge = 0x1p120f;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      f32x16 hit[NRT];
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) hit[rt][r] = 0.f;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const i32x2 w = value_codes(it, vt, tok0, blk, db, std::true_type{});
        bf16x8 nan, vis;
#pragma unroll
        for (int k = 0; k < 8; ++k) nan[k] = (__bf16)(((unsigned)w[k >> 2] >> (8 * (k & 3)) & 0x7f) == 0x7f ? kHuge : 0.f);
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt) {
#pragma unroll
          for (int k = 0; k < 8; ++k) vis[k] = (__bf16)(tok0 + 16 * blk + 8 * h + k < it.sees + row_member[rt] ? kHuge : 0.f);
          hit[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(nan, vis, hit[rt], 0, 0, 0);
        }
      }
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
        for (int r = 0; r < 16; ++r) it.acc[rt][db][r] = __builtin_fmaf(hit[rt][r], 0.f, it.acc[rt][db][r]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // One 32-token tile against the first RT row tiles of the item.
  auto compute_tile = [&](Item& it, const KT& kt, const VT& vt, int ti, auto row_tiles, auto ragged) {
    constexpr bool RAGGED = decltype(ragged)::value;
    constexpr int RT = decltype(row_tiles)::value;
    const int tok0 = ti * kTile;
    float ks[2], vs[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int b = min(2 * ti + blk, it.nblk - 1);
      ks[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(it.ks), b));
      vs[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_scale.y), b));
    }
    f32x16 sr[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r) sr[rt][r] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const i32x4 w = kt.k[i >> 1];
      const bf16x8 a = (i & 1) ? fp8x8_to_bf16(w[2], w[3]) : fp8x8_to_bf16(w[0], w[1]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sr[rt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qreg[rt][i], sr[rt], 0, 0, 0);
    }
    bf16x8 pb[NRT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      // register r holds token 16 * (r / 8) + 8 * h + r % 8 of the tile
      if constexpr (RAGGED) {
        // every score register of a lane belongs to the lane's own query row
        const int row_lim = it.sees > 0 ? min(it.tok_len, it.sees + row_member[rt]) : it.tok_len;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (tok0 + 16 * (r >> 3) + 8 * h + (r & 7) >= row_lim) sr[rt][r] = -INFINITY;
      }
      float mx[2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        mx[blk] = sr[rt][8 * blk];
#pragma unroll
        for (int r = 1; r < 8; ++r) mx[blk] = fmaxf(mx[blk], sr[rt][8 * blk + r]);
      }
      // the scales are positive, so the maximum of the scaled scores is a scaled maximum.  The
      // reference of the exponentials moves (and the accumulators are rescaled) only when a row's
      // maximum rises more than kRescaleSlack above it.
      float mtile = fmaxf(mx[0] * ks[0], mx[1] * ks[1]);
      mtile = fmaxf(mtile, other_half(mtile));
      if (ti == 0) it.mrow[rt] = mtile;
      if (__ballot(mtile > it.mrow[rt] + kRescaleSlack) != 0) {
        const float mnew = fmaxf(it.mrow[rt], mtile);
        const float alpha = fast_exp2(it.mrow[rt] - mnew);
        it.lrow[rt] *= alpha;
        it.mrow[rt] = mnew;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) it.acc[rt][db][r] *= alpha;
      }
      const float mref = it.mrow[rt];
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float e = fast_exp2(__builtin_fmaf(sr[rt][r], ks[r >> 3], -mref));
        // (a masked score times a scale of zero is no number)
        if (RAGGED && sr[rt][r] == -INFINITY) e = 0.f;
        sum += e;
        pb[rt][r >> 3][r & 7] = (__bf16)(e * vs[r >> 3]);
      }
      it.lrow[rt] += sum;
    }
    weighted_values(it, vt, tok0, pb, row_tiles, ragged);
    if constexpr (RAGGED) {
      if (it.sees > 0 && __ballot(holds_nan(vt)) != 0) seen_nans(it, vt, tok0);
    }
  };
  using OneTile = std::integral_constant<int, 1>;
  using AllTiles = std::integral_constant<int, NRT>;

  // Write the partial of the item just attended: live rows go to their places (`to_row` of a row of
  // the tile), through a wave-private strip of LDS so that they leave as whole rows.
  auto write_partial = [&](Item& it, bool two, int live_rows, auto to_row, auto tag_of) {
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      if (rt > 0 && !two) continue;
      const float l = it.lrow[rt] + other_half(it.lrow[rt]);
      // an item half of which nobody attended here (the other wave of the pair took all of it)
      // leaves an empty partial: log-sum-exp -inf, weight 0 in the merge
      const float inv = l == 0.f ? 0.f : 1.f / l;
      stage_partial_row<D, STREAM>(strip, rt * 32 + m, h, it.acc[rt], inv, to_row(rt), (it.mrow[rt] + fast_log2(l)) * kLn2,
                                   p.partial_lse, l != l ? kNanTag : tag_of(rt));
    }
    __builtin_amdgcn_wave_barrier();
    store_partial_rows<D, STREAM>(strip, live_rows, lane, p.partial_out);
    __builtin_amdgcn_wave_barrier();
  };

  bool to_pair_item = false;
  for (int round = 0;; ++round) {
    Item it;
    begin_item(it);
    const int mcnt = __builtin_amdgcn_readfirstlane(r1.x);
    const int ord = __builtin_amdgcn_readfirstlane(r1.y);
    const bool two = NRT > 1 && mcnt * G > 32;
    const int nblk = it.nblk;
    const int ntiles = (it.tok_len + kTile - 1) / kTile;
    const int last = ntiles - 1;
    const int ngroups = (ntiles + 1) >> 1;
    const int a_len = __builtin_amdgcn_readfirstlane(a0.z);
    const int a_nblk = (a_len + kBlock - 1) / kBlock;
    const int a_last = (a_len + kTile - 1) / kTile - 1;
    // first tiles of the next item: its first two, or, for the wave that takes its pair's item from
    // the back, its last two
    const bool a_from_back = Tune::kCoop && coop_back && ta < coop && a_last >= 2 * kCoopMinPairs - 2;
    const int a_t0 = a_from_back ? (a_last & ~1) : 0;

    // ---- all pairs of tiles but the last: every tile full, refills from this item (a refill past the
    // end repeats the last tile so that the number of loads in flight never varies)
    auto stream = [&](auto row_tiles) {
      for (int gr = 0; gr < ngroups - 1; ++gr) {
        const int ti = 2 * gr;
        compute_tile(it, kb0, vb0, ti, row_tiles, std::false_type{});
        load_tile(kb0, vb0, my_blk, nblk, kvh, ti + 2);
        compute_tile(it, kb1, vb1, ti + 1, row_tiles, std::false_type{});
        load_tile(kb1, vb1, my_blk, nblk, kvh, min(ti + 3, last));
      }
    };
    if (NRT == 1 || two) stream(AllTiles{});
    else stream(OneTile{});

    // ---- one step for each of the items ahead: scales (and query rows) of the next, block ids and
    // members of the one after it, record of the third, ticket of the fourth
    int b_blk, b_seq[NRT];
    load_lane_meta(b0, b1, b_blk, b_seq);
    const int tc = resolve_ticket(round + 3);
    int4 c0, c1;
    int ckvh;
    load_record(tc, c0, c1, ckvh);
    issue_ticket(round + 4);
    if constexpr (Tune::kEarlyQ) load_q(nq, a_seq, a1.x, akvh);
    next_scale = load_scales(a_blk, akvh);

    // ---- the last pair, with masks; refills come from the next item (of a ticket past the end: from the
    // last record of the list, loads nobody uses)
    const int ti = 2 * (ngroups - 1);
    compute_tile(it, kb0, vb0, ti, AllTiles{}, std::true_type{});
    load_tile(kb0, vb0, a_blk, a_nblk, akvh, a_t0);
    if (ti + 1 <= last) compute_tile(it, kb1, vb1, ti + 1, AllTiles{}, std::true_type{});
    if constexpr (!Tune::kEarlyQ) load_q(qreg, a_seq, a1.x, akvh);
    // (before the last refill: stores count as outstanding memory operations too)
    write_partial(
        it, two, mcnt * G,
        [&](int rt) -> int64_t {
          return row_member[rt] < mcnt ? ((int64_t)seq[rt] * p.max_partials + ord) * p.num_q_heads + kvh * G + row_head[rt] : -1;
        },
        [](int) { return 0; });
    load_tile(kb1, vb1, a_blk, a_nblk, akvh, min(a_t0 + 1, a_last));

    // ---- move on
    if (ta >= ntickets) break;
    if constexpr (Tune::kEarlyQ) {
#pragma unroll
      for (int i = 0; i < KS; ++i) qreg[0][i] = nq[0][i];
    }
    my_scale = next_scale;
    r0 = a0, r1 = a1, kvh = akvh, my_blk = a_blk;
    a0 = b0, a1 = b1, akvh = bkvh, a_blk = b_blk;
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) seq[rt] = a_seq[rt], a_seq[rt] = b_seq[rt];
    b0 = c0, b1 = c1, bkvh = ckvh;
    t_cur = ta;
    ta = tb;
    tb = tc;
    if (Tune::kCoop && t_cur < coop) {
      to_pair_item = true;
      break;
    }
  }

  // ---- the item shared with the other wave of the pair, the last one of both: pairs of tiles are
  // claimed from a counter of the pair, one wave from the front and one from the back (see
  // fca_attend32.hip for the protocol).
  if (Tune::kCoop && to_pair_item) {
    Item it;
    begin_item(it);
    const int mcnt = __builtin_amdgcn_readfirstlane(r1.x);
    const int ord = __builtin_amdgcn_readfirstlane(r1.y);
    const bool two = NRT > 1 && mcnt * G > 32;
    const int nblk = it.nblk;
    const int ntiles = (it.tok_len + kTile - 1) / kTile;
    const int last = ntiles - 1;
    const int ngroups = (ntiles + 1) >> 1;
    const bool shared_item = ngroups >= kCoopMinPairs;
    if (shared_item || !coop_back) {
      const bool from_back = shared_item && coop_back;
      const int inc = shared_item ? (coop_back ? 1 << 10 : 1) : 0;
      int* ctr = p.coop_ctr + pair_id;
      int added = 0, claim_v = 0;
      auto issue_claim = [&](int by) {
        if (lane == 0) claim_v = atomicAdd(ctr + opaque_zero, by);
        added += by;
      };
      // the pair of tiles after `cur`, or -1 when there is none left for this wave
      auto next_pair = [&](int cur) -> int {
        if (!shared_item) return cur + 1 < ngroups ? cur + 1 : -1;
        const int old = __builtin_amdgcn_readfirstlane(claim_v);
        const int f = old & 1023, b = (old >> 10) & 1023;
        if ((old >> 20) != 0 || 4 + f + b >= ngroups) return -1;
        return coop_back ? ngroups - 3 - b : 2 + f;
      };
      auto compute_any = [&](const KT& kt, const VT& vt, int ti) {
        if (ti > last) return;
        compute_tile(it, kt, vt, ti, AllTiles{}, std::true_type{});
      };
      int cur = from_back ? ngroups - 1 : 0;
      int nxt = from_back ? ngroups - 2 : (ngroups > 1 ? 1 : -1);  // granted
      issue_claim(inc);
      for (;;) {
        const int refill = nxt >= 0 ? nxt : cur;  // (past the end: loads nobody uses, as above)
        compute_any(kb0, vb0, 2 * cur);
        load_tile(kb0, vb0, my_blk, nblk, kvh, 2 * refill);
        compute_any(kb1, vb1, 2 * cur + 1);
        load_tile(kb1, vb1, my_blk, nblk, kvh, min(2 * refill + 1, last));
        if (nxt < 0) break;
        cur = nxt;
        nxt = next_pair(cur);
        issue_claim(nxt >= 0 ? inc : 0);
      }
      const int back_row = pair_id * (32 * NRT) + m;
      write_partial(
          it, two, mcnt * G,
          [&](int rt) -> int64_t {
            if (row_member[rt] >= mcnt) return -1;
            return from_back ? p.coop_row0 + back_row + 32 * rt
                             : ((int64_t)seq[rt] * p.max_partials + ord) * p.num_q_heads + kvh * G + row_head[rt];
          },
          // the front partial says where the back partial of the same query row is
          [&](int rt) { return shared_item && !coop_back ? 32 + back_row + 32 * rt : 0; });
      if (shared_item && lane == 0) atomicAdd(ctr, (coop_back ? -(1 << 20) : (1 << 20)) - added);
    }
  }
  // loads nobody uses are still in flight: let them land before the wave ends
  __builtin_amdgcn_s_waitcnt(0);
}

hipError_t launch_attend_block(const AttendParams& p, const fca_plan& plan, int max_workgroups, hipStream_t stream) {
  const MetaLayout L = make_layout(plan);
  const int64_t max_tickets = L.max_items * plan.num_kv_heads;
  int grid = 256 * (plan.head_dim == 64 ? 2 : 1);
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
