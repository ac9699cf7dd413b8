// Forest cascade attention over the block-scaled 8-bit cache (fca_block_scales.h): the work items,
// tile orders, matrix products and partial rows of the per-head fp8 kernels (fca_attend.hip), with
// a K scale and a V scale per block of 16 tokens.
//
//   S[t, row] = softmax_scale * s_k[block of t] * sum_d c_k[t, d] q[row, d]
//   O[d, row] = sum_t c_v[d, t] * (s_v[block of t] * P[t, row])
//
// A 32-token tile covers two blocks, and the accumulator registers 0-7 and 8-15 of a lane hold the
// tokens of the first and the second: the K scale is one of two wave-uniform factors of the
// exponent's fused multiply-add, the V scale one factor of a probability before it is rounded to a
// half for the value product (see RowState).  The codes go through the matrix cores as bf16 (K, next to
// bf16 query rows) and as halves (V), both of which hold every e4m3 value exactly.
// (As codes, with the query row split into two rows of codes, a product is no faster, and the 8-bit
// matrix instructions drop products below 2^-13 of the largest one they add.)
//
// Memory-bound where the cache is long: 64 x 8 sequences over prompts of 2560 tokens and 512 of their
// own (32 query heads, 8 KV heads of 128; 913 MB of codes) take 163 us = 5.6 TB/s, a copy of the kernel
// that only loads 153; one sequence of 131071 tokens 46 us = 5.9 TB/s.  Latency-bound where it is short:
// one sequence of 300 tokens takes 8.4 us, five dependent trips to memory from the header to the rows.
#include <hip/hip_ext.h>

#include <type_traits>

#include "fca_attend_block.h"

namespace fca {

// Workgroups per CU: a wave's registers are 512 / this.
template <int D>
constexpr int block_workgroups() { return D == 64 ? 2 : 1; }

template <int D, bool STREAM>
__global__ __launch_bounds__(kThreads, block_workgroups<D>()) void fca_attend_block_kernel(AttendParams p) {
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

  // row m of the stacked query tile is (member m / G, head m % G)
  const int row_member = m / G, row_head = m - row_member * G;
  // MFMA row m carries the token whose index has bits 2 and 3 of m swapped: the score
  // accumulator then holds, per lane half, tokens 8h..8h+7 of each block in register order.
  const int tok_of_m = (m & 3) | ((m & 4) << 1) | ((m & 8) >> 1);
  const int k_lane_off = h * 256 + tok_of_m * 16;
  const int v_lane_off = (h * 32 + m) * 16;  // channel 32 * (2 * pair + h) + m, all 16 tokens
  // wave-private strip of LDS for the output rows
  __shared__ __attribute__((aligned(16))) char strips[kWaves][32 * strip_row_bytes<D>()];
  char* strip = strips[wave];
  const float2* scales = reinterpret_cast<const float2*>(p.k_scale);

  // Dealing the work, as in fca_attend32.hip: the largest tickets go one to a pair of waves on
  // different XCDs, which take them last and from both ends; the rest is dealt back and forth over
  // the size-ordered list, and its last full round and remainder are drawn from a counter.
  const int half_grid = (int)gridDim.x >> 1;
  const bool coop_back = (int)blockIdx.x >= half_grid;
  const int pair_id = (coop_back ? (((int)blockIdx.x ^ 3) - half_grid) : (int)blockIdx.x) * kWaves + wave;
  constexpr bool COOP = block_workgroups<D>() == 1;
  const bool coop_on = COOP && p.coop_ctr != nullptr && (gridDim.x & 7) == 0 && nwaves / 2 <= p.coop_pairs &&
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
  auto load_lane_meta = [&](const int4& r0, const int4& r1, int& my_blk, int& seq) {
    const int nblk = (r0.z + kBlock - 1) / kBlock;
    my_blk = p.block_table[(int64_t)r0.x * p.bt_stride + r0.y + min(lane, nblk - 1)];
    seq = meta[p.off_members + r0.w + (row_member < r1.x ? row_member : 0)];
  };
  // ... and off the block ids: the scales of the lane's block
  auto load_scales = [&](int my_blk, int kvh) -> float2 { return scales[(int64_t)my_blk * Hkv + kvh]; };
  auto load_q = [&](bf16x8 (&q)[KS], int seq, int mcnt, int kvh) {
    const bool live = row_member < mcnt;
    const __bf16* qp = reinterpret_cast<const __bf16*>(p.q) + (int64_t)seq * p.q_seq_stride + (int64_t)(kvh * G + row_head) * p.q_head_stride;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      // the K tile hands a lane 16 channels of one token: two steps
      bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
      if (!live) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
      q[i] = v;
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
  int my_blk, a_blk, seq, a_seq;
  int t_cur = resolve_ticket(0);  // rounds 0 to 3 are static, or the whole list is
  int ta = resolve_ticket(1);
  int tb = resolve_ticket(2);
  load_record(t_cur, r0, r1, kvh);
  load_record(ta, a0, a1, akvh);
  load_record(tb, b0, b1, bkvh);
  load_lane_meta(r0, r1, my_blk, seq);
  load_lane_meta(a0, a1, a_blk, a_seq);
  bf16x8 qreg[KS], nq[KS];
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
    f32x16 acc[NDB];
    RowState row;
    float ks;  // K scale of the lane's block, times softmax scale and log2(e)
    float lv;  // log2 of its V scale
  };
  auto begin_item = [&](Item& it) {
    it.tok_len = __builtin_amdgcn_readfirstlane(r0.z);
    it.nblk = (it.tok_len + kBlock - 1) / kBlock;
    it.sees = __builtin_amdgcn_readfirstlane(r1.w);
    it.ks = my_scale.x * (p.scale * kLog2e);
    it.lv = scale_log2(my_scale.y);
    it.row = empty_row();
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) it.acc[db][r] = 0.f;
  };

  // One 32-token tile.  RAGGED: it may run past the end of the chunk, or past what a row sees.
  auto compute_tile = [&](Item& it, const KT& kt, const VT& vt, int ti, auto ragged) {
    constexpr bool RAGGED = decltype(ragged)::value;
    const int tok0 = ti * kTile;
    float ks[2], vs[2], lv[2];
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const int b = min(2 * ti + blk, it.nblk - 1);
      ks[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(it.ks), b));
      vs[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_scale.y), b));
      lv[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(it.lv), b));
    }
    f32x16 sr;
#pragma unroll
    for (int r = 0; r < 16; ++r) sr[r] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const i32x4 w = kt.k[i >> 1];
      const bf16x8 a = (i & 1) ? fp8x8_to_bf16(w[2], w[3]) : fp8x8_to_bf16(w[0], w[1]);
      sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qreg[i], sr, 0, 0, 0);
    }
    const int lim = (it.sees > 0 ? min(it.tok_len, it.sees + row_member) : it.tok_len) - tok0 - 8 * h;
    f16x8 pb[2];  // weights of the tile as B operands
    weigh_tile<RAGGED>(it.row, ti == 0, sr, ks, vs, lv, lim, it.acc, pb);
    // (`run`: the last tile of a query run, whose rows see different numbers of its tokens)
    const bool run = RAGGED && it.sees > 0;
    int nans = 0;
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int pair = 0; pair < NDB / 2; ++pair) {
        i32x4 raw = vt.v[blk][pair];
        if constexpr (RAGGED) {
          raw = first_codes(raw, it.tok_len - (tok0 + 16 * blk));
          if (run) raw = without_nans(raw, nans);
        }
#pragma unroll
        for (int db = 2 * pair; db < 2 * pair + 2; ++db) {
          const i32x2 w = value_codes(raw, db);
          it.acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp8x8_to_f16(w), pb[blk], it.acc[db], 0, 0, 0);
        }
      }
    // A NaN among the values of such a tile must not reach the rows that do not see its token (0 * NaN),
    // so it was left out of the product.  Where a row does see one, the product of (huge where the
    // value is NaN) and (huge where the row sees the token) overflows, and infinity * 0 makes the row's
    // sum of that channel NaN.
    if constexpr (RAGGED) {
      if (__ballot(nans != 0) != 0) {
        const int seen = it.sees + row_member - tok0 - 8 * h;  // tokens of the lane's eight, block 0
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          f32x16 hit;
#pragma unroll
          for (int r = 0; r < 16; ++r) hit[r] = 0.f;
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            const i32x2 w = value_codes(first_codes(vt.v[blk][db >> 1], it.tok_len - (tok0 + 16 * blk)), db);
            bf16x8 vis;
#pragma unroll
            for (int k = 0; k < 8; ++k) vis[k] = (__bf16)(k + 16 * blk < seen ? kHuge : 0.f);
            hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(huge_at_nans(w), vis, hit, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) it.acc[db][r] = __builtin_fmaf(hit[r], 0.f, it.acc[db][r]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };

  // Write the partial of the item just attended: live rows go to `prow` (-1: a dead row), through a
  // wave-private strip of LDS so that they leave as whole rows; `tag` rides in the row's scale.
  auto write_partial = [&](Item& it, int64_t prow, int live_rows, int tag) {
    const float l = it.row.l + other_half(it.row.l);
    // an item half of which nobody attended here (the other wave of the pair took all of it)
    // leaves an empty partial: log-sum-exp -inf, weight 0 in the merge
    const float inv = l == 0.f ? 0.f : 1.f / l;
    stage_partial_row<D, STREAM>(strip, m, h, it.acc, inv / it.row.g, prow, (it.row.m + fast_log2(l)) * kLn2, p.partial_lse, l != l ? kNanTag : tag);
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
    const int nblk = it.nblk;
    const int ntiles = (it.tok_len + kTile - 1) / kTile;
    const int last = ntiles - 1;
    const int ngroups = (ntiles + 1) >> 1;
    const int a_len = __builtin_amdgcn_readfirstlane(a0.z);
    const int a_nblk = (a_len + kBlock - 1) / kBlock;
    const int a_last = (a_len + kTile - 1) / kTile - 1;
    // first tiles of the next item: its first two, or, for the wave that takes its pair's item from
    // the back, its last two
    const bool a_from_back = COOP && coop_back && ta < coop && a_last >= 2 * kCoopMinPairs - 2;
    const int a_t0 = a_from_back ? (a_last & ~1) : 0;

    // ---- all pairs of tiles but the last: every tile full, refills from this item (a refill past the
    // end repeats the last tile so that the number of loads in flight never varies)
    for (int gr = 0; gr < ngroups - 1; ++gr) {
      const int ti = 2 * gr;
      compute_tile(it, kb0, vb0, ti, std::false_type{});
      load_tile(kb0, vb0, my_blk, nblk, kvh, ti + 2);
      compute_tile(it, kb1, vb1, ti + 1, std::false_type{});
      load_tile(kb1, vb1, my_blk, nblk, kvh, min(ti + 3, last));
    }

    // ---- one step for each of the items ahead: scales (and query rows) of the next, block ids and
    // members of the one after it, record of the third, ticket of the fourth
    int b_blk, b_seq;
    load_lane_meta(b0, b1, b_blk, b_seq);
    const int tc = resolve_ticket(round + 3);
    int4 c0, c1;
    int ckvh;
    load_record(tc, c0, c1, ckvh);
    issue_ticket(round + 4);
    load_q(nq, a_seq, a1.x, akvh);
    next_scale = load_scales(a_blk, akvh);

    // ---- the last pair, with masks; refills come from the next item (of a ticket past the end: from the
    // last record of the list, loads nobody uses)
    const int ti = 2 * (ngroups - 1);
    compute_tile(it, kb0, vb0, ti, std::true_type{});
    load_tile(kb0, vb0, a_blk, a_nblk, akvh, a_t0);
    if (ti + 1 <= last) compute_tile(it, kb1, vb1, ti + 1, std::true_type{});
    // (before the last refill: stores count as outstanding memory operations too)
    write_partial(it, row_member < mcnt ? ((int64_t)seq * p.max_partials + ord) * p.num_q_heads + kvh * G + row_head : -1, mcnt * G, 0);
    load_tile(kb1, vb1, a_blk, a_nblk, akvh, min(a_t0 + 1, a_last));

    // ---- move on
    if (ta >= ntickets) break;
#pragma unroll
    for (int i = 0; i < KS; ++i) qreg[i] = nq[i];
    my_scale = next_scale;
    r0 = a0, r1 = a1, kvh = akvh, my_blk = a_blk, seq = a_seq;
    a0 = b0, a1 = b1, akvh = bkvh, a_blk = b_blk, a_seq = b_seq;
    b0 = c0, b1 = c1, bkvh = ckvh;
    t_cur = ta;
    ta = tb;
    tb = tc;
    if (COOP && t_cur < coop) {
      to_pair_item = true;
      break;
    }
  }

  // ---- the item shared with the other wave of the pair, the last one of both: pairs of tiles are
  // claimed from a counter of the pair, one wave from the front and one from the back (see
  // fca_attend32.hip for the protocol).
  if (COOP && to_pair_item) {
    Item it;
    begin_item(it);
    const int mcnt = __builtin_amdgcn_readfirstlane(r1.x);
    const int ord = __builtin_amdgcn_readfirstlane(r1.y);
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
        compute_tile(it, kt, vt, ti, std::true_type{});
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
      const int back_row = pair_id * 32 + m;
      const int64_t row = from_back ? p.coop_row0 + back_row : ((int64_t)seq * p.max_partials + ord) * p.num_q_heads + kvh * G + row_head;
      // the front partial says where the back partial of the same query row is
      write_partial(it, row_member < mcnt ? row : -1, mcnt * G, shared_item && !coop_back ? 32 + back_row : 0);
      if (shared_item && lane == 0) atomicAdd(ctr, (coop_back ? -(1 << 20) : (1 << 20)) - added);
    }
  }
  // loads nobody uses are still in flight: let them land before the wave ends
  __builtin_amdgcn_s_waitcnt(0);
}

static int compute_units() {
  static const int cus = [] {
    int dev = 0, n = 0;
    const bool known = hipGetDevice(&dev) == hipSuccess &&
                       hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0;
    return known ? n : 256;
  }();
  return cus;
}

hipError_t launch_attend_block(const AttendParams& p, const fca_plan& plan, int max_workgroups, hipStream_t stream) {
  if (plan.rows_per_item == 64 || plan.head_dim == 256)
    return launch_attend_block_wide(p, plan, compute_units(), max_workgroups, stream);
  const MetaLayout L = make_layout(plan);
  const int64_t max_tickets = L.max_items * plan.num_kv_heads;
  int grid = compute_units() * (plan.head_dim == 64 ? block_workgroups<64>() : block_workgroups<128>());
  // the caller's cap: leaves CUs to other streams
  if (max_workgroups > 0 && max_workgroups < grid) grid = max_workgroups;
  if ((int64_t)grid * kWaves > max_tickets) grid = (int)((max_tickets + kWaves - 1) / kWaves);
  if (grid < 1) grid = 1;
  // With sharing on, and but for query runs, a launch reads every KV block about once: past the caches.
  const bool stream_kv = plan.max_levels > 0 && !p.kv_reread;
  hipEvent_t ev_start, ev_stop;
  take_attend_timing(&ev_start, &ev_stop);
#define FCA_LAUNCH(D_, S_) \
  if (ev_start) hipExtLaunchKernelGGL((fca_attend_block_kernel<D_, S_>), dim3(grid), dim3(kThreads), 0, stream, ev_start, ev_stop, 0, p); \
  else hipLaunchKernelGGL((fca_attend_block_kernel<D_, S_>), dim3(grid), dim3(kThreads), 0, stream, p)
#define FCA_PICK(D_) \
  if (stream_kv) { FCA_LAUNCH(D_, true); } else { FCA_LAUNCH(D_, false); }
  if (plan.head_dim == 128) {
    FCA_PICK(128);
  } else {
    FCA_PICK(64);
  }
#undef FCA_PICK
#undef FCA_LAUNCH
  return hipGetLastError();
}

}  // namespace fca
