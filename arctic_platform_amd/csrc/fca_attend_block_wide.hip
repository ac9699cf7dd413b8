// Forest cascade attention over the block-scaled cache where one wave's registers are too few: items
// of 64 query rows (head sizes 64 and 128) and head size 256.
//
// The work items, tile orders and partial rows are those of fca_attend_block.hip; here a workgroup
// of two waves attends an item together.  With 64 rows each wave takes 32 of them, at head size 256
// each takes half of the output channels (and forms all scores).  Both need every tile of K and V,
// and a wave that keeps two row tiles, its query rows and tiles in flight in registers has too few
// bytes in flight: it measured 1.77 us per 8 KB tile where memory delivers one in 1.36.  So the tiles
// go through a ring of LDS slots filled by direct-to-LDS loads, which needs no landing registers: the
// ring runs kAhead tiles in front of the arithmetic, over item boundaries too, and a wave stays below
// 256 registers, so that two share a SIMD and one computes while the other waits.
//
// One barrier per tile: a wave waits for its own requests of the tile about to be used (each wave
// requests half a tile; loads complete in order), and behind the barrier everyone's have landed and
// everyone has finished with the tile before, whose slot the next request refills.
//
// Measured (32 query heads, 8 KV heads of 128): 16 x 6 sequences of four query tokens over 1500 + 400
// tokens 48 us; 8 x 16 over 32768 + 2176 tokens 240 us = 4.7 TB/s, of which the partial rows are 20 (only
// loading takes 187); 16 query heads on 2 KV heads of 256, 32 x 8 over 2560 + 512 tokens, 69 us.  What
// bounds it: a wave issues for about 1100 cycles a tile (250 vector and 16 matrix instructions), two
// share a SIMD and a tile takes a workgroup 0.93 us; an item adds 1 us, the start of a launch 6 to 8
// (header, records, block ids and query rows are dependent trips to memory, all workgroups at once).
// Sharing the last items between pairs of workgroups evened their ends out and made no launch faster:
// a workgroup that is done leaves its issue slots to its neighbours.
#include <hip/hip_ext.h>

#include <type_traits>

#include "fca_attend_block.h"

namespace fca {

// Direct-to-LDS loads: a wave copies `PIECES` KB of a block to LDS as they lie.  An instruction moves 16
// bytes per lane to M0 + 16 * lane, and its immediate offset counts on both sides.  Written as assembly so
// that the compiler's wait insertion does not know of the loads (it would drain them before every LDS
// read); loads it does not know of only make its own waits more conservative.  Nor does its hazard
// check look inside: a load to LDS follows a write of M0, and of a scalar register by a vector
// instruction, by at least one and five wait states, which the s_nop provides.
__device__ inline unsigned lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((unsigned)(size_t)((__attribute__((address_space(3))) void*)(p)));
}
template <int PIECES, bool STREAM>
__device__ inline void block_to_lds(const char* block, int lane_off, unsigned lds) {
  static_assert(PIECES == 1 || PIECES == 2 || PIECES == 4, "");
#define FCA_TO_LDS(MORE, NT) \
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" NT MORE : : "v"(lane_off), "s"(block), "s"(lds) : "memory", "m0")
#define FCA_PIECE(OFF, NT) "\n\tglobal_load_lds_dwordx4 %0, %1 offset:" OFF NT
  if constexpr (STREAM) {
    if constexpr (PIECES == 1) FCA_TO_LDS("", " nt");
    if constexpr (PIECES == 2) FCA_TO_LDS(FCA_PIECE("1*1024", " nt"), " nt");
    if constexpr (PIECES == 4) FCA_TO_LDS(FCA_PIECE("1*1024", " nt") FCA_PIECE("2*1024", " nt") FCA_PIECE("3*1024", " nt"), " nt");
  } else {
    if constexpr (PIECES == 1) FCA_TO_LDS("", "");
    if constexpr (PIECES == 2) FCA_TO_LDS(FCA_PIECE("1*1024", ""), "");
    if constexpr (PIECES == 4) FCA_TO_LDS(FCA_PIECE("1*1024", "") FCA_PIECE("2*1024", "") FCA_PIECE("3*1024", ""), "");
  }
#undef FCA_PIECE
#undef FCA_TO_LDS
}
// s_waitcnt that constrains only the vector-memory counter (gfx9 encoding)
#define FCA_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt(0x0f70 | ((n) & 15) | (((n) >> 4) << 14))

template <int D>
struct WideTuning {
  static constexpr bool kChannels = D == 256;            // the waves split channels instead of rows
  static constexpr int kWaveD = kChannels ? D / 2 : D;   // output channels of a wave
  static constexpr int kWorkgroups = kChannels ? 3 : 4;  // per CU (160 KB of LDS)
  static constexpr int kSlots = kChannels ? 3 : 4;
  static constexpr int kAhead = kSlots - 1;
  static constexpr int kBlockPieces = D / 64;            // 1 KB pieces of a block's K or V
  static constexpr int kSlotBytes = 4 * D * kBlock;      // a tile: K of its two blocks, V of its two blocks
  static constexpr bool kEarlyQ = !kChannels;            // the next item's query rows are fetched an item ahead
};

template <int D, bool STREAM>
__global__ __launch_bounds__(128, 2) void fca_attend_block_wide_kernel(AttendParams p) {
  using Tune = WideTuning<D>;
  constexpr int KS = D / 16;              // MFMA steps of the score product
  constexpr int NDB = Tune::kWaveD / 32;  // 32-channel blocks of a wave's output
  constexpr int NK = D / 32, NI = D / 32; // pieces of K; pieces a wave requests per tile
  constexpr int kAhead = Tune::kAhead;

  __shared__ __attribute__((aligned(16))) char ring[Tune::kSlots][Tune::kSlotBytes];
  __shared__ float row_amax[2][32];

  const int32_t* hdr = p.meta + p.off_header;
  const int total = hdr[H_ITEMS], shared = hdr[H_SHARED_ITEMS];
  const int first = p.select == 2 ? shared : 0;
  const int last_item = p.select == 1 ? shared : total;
  const int ntickets = (last_item - first) * p.num_kv_heads;
  const int nwg = (int)gridDim.x, me = (int)blockIdx.x;
  if (me >= ntickets) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m = lane & 31, h = lane >> 5;
  const int G = p.group, Hkv = p.num_kv_heads;
  const int32_t* meta = p.meta;
  const float2* scales = reinterpret_cast<const float2*>(p.k_scale);
  const unsigned ring_lds = lds_address(&ring[0][0]);

  // Row `row_tile * 32 + m` of the stacked query tile is (member row / G, head row % G).  Which wave
  // takes which row tile changes from item to item: an item of 32 rows or fewer has work for one of
  // the two, and that must not always be a wave on the same SIMD.
  auto tile_of = [&](int round) { return Tune::kChannels ? 0 : (wave + round + me) & 1; };
  const int member_of[2] = {m / G, (32 + m) / G};
  const int head_of[2] = {m - member_of[0] * G, 32 + m - member_of[1] * G};
  const int channel0 = Tune::kChannels ? wave * Tune::kWaveD : 0;  // first output channel of this wave
  // MFMA row m carries the token whose index has bits 2 and 3 of m swapped: the score accumulator then
  // holds, per lane half, tokens 8h..8h+7 of each block in register order.
  const int tok_of_m = (m & 3) | ((m & 4) << 1) | ((m & 8) >> 1);
  const int k_off = (m >> 4) * D * kBlock + h * 256 + tok_of_m * 16;  // of a lane's codes in a tile
  const int v_off = 2 * D * kBlock + (channel0 + m) * kBlock + h * 8;
  // wave 0 requests K, wave 1 V
  const char* plane = wave == 0 ? p.k_cache : p.v_cache;

  // Every ticket is dealt in advance: back and forth over the size-ordered list.
  auto ticket = [&](int r) { return r * nwg + ((r & 1) ? nwg - 1 - me : me); };
  // An item record, in scalar registers; one in flight is kept as it was loaded.
  struct Item {
    int rep, blk_start, tok_len, members, mcnt, ord, sees, kvh;
  };
  struct RawItem {
    int4 r0, r1;  // rep, blk_start, tok_len, member_off; member_cnt, ord, node, sees
    int kvh;
  };
  auto load_record = [&](int t) {
    const int tc = min(t, ntickets - 1);  // (a ticket past the end reads a valid record)
    const int it = tc / Hkv;
    const int4* rec = reinterpret_cast<const int4*>(meta + p.off_items + (int64_t)(first + it) * kItemInts);
    return RawItem{rec[0], rec[1], tc - it * Hkv};
  };
  auto arrived = [&](const RawItem& c) {
    return Item{__builtin_amdgcn_readfirstlane(c.r0.x), __builtin_amdgcn_readfirstlane(c.r0.y), __builtin_amdgcn_readfirstlane(c.r0.z),
                __builtin_amdgcn_readfirstlane(c.r0.w), __builtin_amdgcn_readfirstlane(c.r1.x), __builtin_amdgcn_readfirstlane(c.r1.y),
                __builtin_amdgcn_readfirstlane(c.r1.w), c.kvh};
  };
  auto blocks_of = [](const Item& x) { return (x.tok_len + kBlock - 1) / kBlock; };
  auto tiles_of = [](const Item& x) { return (x.tok_len + kTile - 1) / kTile; };
  // one block id of the chunk per lane (a chunk has at most 64 blocks) and the member sequence of this
  // lane's query row
  auto load_lane_meta = [&](const Item& x, int row_tile, int& blk, int& seq) {
    const int row_member = row_tile ? member_of[1] : member_of[0];
    blk = p.block_table[(int64_t)x.rep * p.bt_stride + x.blk_start + min(lane, blocks_of(x) - 1)];
    seq = meta[p.off_members + x.members + (row_member < x.mcnt ? row_member : 0)];
  };
  auto load_q = [&](bf16x8 (&q)[KS], const Item& x, int row_tile, int seq) {
    const int row_member = row_tile ? member_of[1] : member_of[0], row_head = row_tile ? head_of[1] : head_of[0];
    const bool live = row_member < x.mcnt;
    const __bf16* qp = reinterpret_cast<const __bf16*>(p.q) + (int64_t)seq * p.q_seq_stride + (int64_t)(x.kvh * G + row_head) * p.q_head_stride;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      // the K tile hands a lane 16 channels of one token: two steps
      bf16x8 v = *reinterpret_cast<const bf16x8*>(qp + 32 * (i >> 1) + 16 * h + 8 * (i & 1));
      if (!live) v = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
      q[i] = v;
    }
  };
  // This wave's half of a tile.
  int req_slot = 0;
  auto request = [&](const Item& x, int blk_ids, int ti) {
    const int b0 = __builtin_amdgcn_readlane(blk_ids, 2 * ti);
    const int b1 = __builtin_amdgcn_readlane(blk_ids, min(2 * ti + 1, blocks_of(x) - 1));
    const char* base = plane + (int64_t)x.kvh * p.kv_head_bytes;
    const unsigned to = ring_lds + req_slot * Tune::kSlotBytes + wave * (2 * D * kBlock);
    block_to_lds<Tune::kBlockPieces, STREAM>(base + (int64_t)b0 * p.kv_block_bytes, lane * 16, to);
    block_to_lds<Tune::kBlockPieces, STREAM>(base + (int64_t)b1 * p.kv_block_bytes, lane * 16, to + D * kBlock);
    req_slot = req_slot + 1 == Tune::kSlots ? 0 : req_slot + 1;
  };

  // ---- set-up: records of the first three items, everything else of the first two
  Item cur = arrived(load_record(ticket(0))), nxt = arrived(load_record(ticket(1))), third = arrived(load_record(ticket(2)));
  int my_blk, a_blk, seq, a_seq;
  load_lane_meta(cur, tile_of(0), my_blk, seq);
  load_lane_meta(nxt, tile_of(1), a_blk, a_seq);
  bf16x8 qreg[KS], nq[Tune::kEarlyQ ? KS : 1];
  load_q(qreg, cur, tile_of(0), seq);
  float2 my_scale = scales[(int64_t)my_blk * Hkv + cur.kvh];
  // Items take at least kAhead places in the stream of tiles (a short one repeats its last tile, which
  // nobody attends again), so that the ring never runs further ahead than into the next item.
  for (int s = 0; s < kAhead; ++s) request(cur, my_blk, min(s, tiles_of(cur) - 1));
  int slot = 0;

  for (int round = 0;; ++round) {
    // ---- a step for each of the items ahead: query rows and scales of the next, block ids and members
    // of the one after it, record of the third
    int b_blk, b_seq;
    load_lane_meta(third, tile_of(round + 2), b_blk, b_seq);
    const RawItem fourth = load_record(ticket(round + 3));
    if constexpr (Tune::kEarlyQ) load_q(nq, nxt, tile_of(round + 1), a_seq);
    const float2 next_scale = scales[(int64_t)a_blk * Hkv + nxt.kvh];
    // Query rows fetched late have to be here before the loop over the tiles: a wait for them inside it
    // would also wait, every tile, for the requests the compiler does not know of.
    if constexpr (!Tune::kEarlyQ) FCA_WAIT_VMCNT(0);

    const int tok_len = cur.tok_len, mcnt = cur.mcnt;
    // Last chunk of a query-run tile: member i sees the first `sees + i` tokens of the chunk (its own
    // token and what is before it); all members end inside the last tile.
    const int sees = cur.sees;
    const int nblk = blocks_of(cur);
    const int ntiles = tiles_of(cur), last = ntiles - 1, a_last = tiles_of(nxt) - 1;
    const int nfull = (tok_len - (sees > 0 ? 1 : 0)) / kTile;
    const int places = max(ntiles, kAhead);
    const int row_tile = tile_of(round);
    const int row_member = row_tile ? member_of[1] : member_of[0], row_head = row_tile ? head_of[1] : head_of[0];
    const bool has_rows = row_tile == 0 || mcnt * G > 32;
    const float ks_lane = my_scale.x * (p.scale * kLog2e);  // K scale of the lane's block, log2 domain
    const float lv_lane = scale_log2(my_scale.y);

    f32x16 acc[NDB];
    RowState state = empty_row();
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;

    auto compute_tile = [&](int ti, auto ragged) {
      constexpr bool RAGGED = decltype(ragged)::value;
      const int tok0 = ti * kTile;
      float ks[2], vs[2], lv[2];
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const int b = min(2 * ti + blk, nblk - 1);
        ks[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ks_lane), b));
        vs[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_scale.y), b));
        lv[blk] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lv_lane), b));
      }
      // (the fences keep reads of LDS together in front of the arithmetic they feed, V's in front of the
      // softmax: left alone the compiler reads one piece, waits for it, and reads the next)
      i32x4 kw[NK];
      i32x2 vw[2][NDB];
#pragma unroll
      for (int i = 0; i < NK; ++i) kw[i] = *reinterpret_cast<const i32x4*>(&ring[slot][0] + k_off + 512 * i);
      __builtin_amdgcn_sched_barrier(0);
      f32x16 sr;
#pragma unroll
      for (int r = 0; r < 16; ++r) sr[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp8x8_to_bf16(kw[i][0], kw[i][1]), qreg[2 * i], sr, 0, 0, 0);
        sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp8x8_to_bf16(kw[i][2], kw[i][3]), qreg[2 * i + 1], sr, 0, 0, 0);
      }
      // codes of tokens 8h..8h+7 of channel 32 * db + m
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
          vw[blk][db] = *reinterpret_cast<const i32x2*>(&ring[slot][0] + v_off + (blk * D + 32 * db) * kBlock);
      __builtin_amdgcn_sched_barrier(0);
      const int lim = (sees > 0 ? min(tok_len, sees + row_member) : tok_len) - tok0 - 8 * h;
      f16x8 pb[2];  // weights of the tile as B operands
      weigh_tile<RAGGED>(state, ti == 0, sr, ks, vs, lv, lim, acc, pb);
      // (`run`: the last tile of a query run, whose rows see different numbers of its tokens)
      const bool run = RAGGED && sees > 0;
      int nans = 0;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk)
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          i32x2 w = vw[blk][db];
          if constexpr (RAGGED) {
            w = first_codes(w, tok_len - (tok0 + 16 * blk + 8 * h));
            if (run) w = without_nans(w, nans);
          }
          acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp8x8_to_f16(w), pb[blk], acc[db], 0, 0, 0);
        }
      // A NaN among the values of such a tile must not reach the rows that do not see its token (0 * NaN),
      // so it was left out of the product.  Where a row does see one, the product of (huge where the
      // value is NaN) and (huge where the row sees the token) overflows, and infinity * 0 makes the row's
      // sum of that channel NaN.
      if constexpr (RAGGED) {
        if (__ballot(nans != 0) != 0) {
          const int seen = sees + row_member - tok0 - 8 * h;  // tokens of the lane's eight, block 0
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            f32x16 hit;
#pragma unroll
            for (int r = 0; r < 16; ++r) hit[r] = 0.f;
#pragma unroll
            for (int blk = 0; blk < 2; ++blk) {
              const i32x2 w = first_codes(vw[blk][db], tok_len - (tok0 + 16 * blk + 8 * h));
              bf16x8 vis;
#pragma unroll
              for (int k = 0; k < 8; ++k) vis[k] = (__bf16)(k + 16 * blk < seen ? kHuge : 0.f);
              hit = __builtin_amdgcn_mfma_f32_32x32x16_bf16(huge_at_nans(w), vis, hit, 0, 0, 0);
              __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[db][r] = __builtin_fmaf(hit[r], 0.f, acc[db][r]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    };

    auto next_tile = [&](int s) {  // the tile at place s is here; the one kAhead places on is on its way
      FCA_WAIT_VMCNT((kAhead - 1) * NI);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's reads of the slot about to be refilled have returned
      __builtin_amdgcn_s_barrier();
      const int ahead = s + kAhead;
      if (ahead < places) request(cur, my_blk, min(ahead, last));
      else request(nxt, a_blk, min(ahead - places, a_last));
    };
    int s = 0;
    for (; s < nfull; ++s) {
      next_tile(s);
      if (has_rows) compute_tile(s, std::false_type{});
      slot = slot + 1 == Tune::kSlots ? 0 : slot + 1;
    }
    for (; s < places; ++s) {
      next_tile(s);
      if (has_rows && s < ntiles) compute_tile(s, std::true_type{});
      slot = slot + 1 == Tune::kSlots ? 0 : slot + 1;
    }

    // ---- the item's partial rows: normalised, as halves times one power of two per row.  A lane has
    // every other four channels of its row; after a swap with the lane 32 away it has eight adjacent
    // ones.  (Through a strip of LDS, so that rows leave whole, it took 3 us an item.)
    {
      const float l = state.l + other_half(state.l);
      const float inv = 1.f / l / state.g;  // (l * g could overflow where all V scales are small)
      float amax = 0.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) amax = fmaxf(amax, fabsf(acc[db][r]));
      amax = fmaxf(amax, other_half(amax)) * fabsf(inv);
      if constexpr (Tune::kChannels) {  // the row's scale is that of both waves' channels
        if (h == 0) row_amax[wave][m] = amax;
        __syncthreads();
        amax = fmaxf(amax, row_amax[wave ^ 1][m]);
      }
      const float scale = pow2_ceil(amax);
      const float k = inv / scale;  // exact: the scale is a power of two
      const int64_t prow = has_rows && row_member < mcnt ? ((int64_t)seq * p.max_partials + cur.ord) * p.num_q_heads + cur.kvh * G + row_head : -1;
      if (h == 0 && prow >= 0 && (!Tune::kChannels || wave == 0)) {
        const f32x2 ls = {(state.m + fast_log2(l)) * kLn2, __uint_as_float(__float_as_uint(scale) | (l != l ? (unsigned)kNanTag : 0u))};
        if constexpr (STREAM) store8_coherent(p.partial_lse + 2 * prow, __builtin_bit_cast(uint64_t, ls));
        else *reinterpret_cast<f32x2*>(p.partial_lse + 2 * prow) = ls;
      }
      if (has_rows) {
        char* dst = static_cast<char*>(p.partial_out) + (max(prow, (int64_t)0) * D + channel0 + 8 * h) * 2;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            i32x2 v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              f16x4 x;
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = (_Float16)(acc[db][8 * q + 4 * j + e] * k);
              v[j] = __builtin_bit_cast(i32x2, x);
            }
            const auto s0 = __builtin_amdgcn_permlane32_swap((unsigned)v[0][0], (unsigned)v[1][0], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap((unsigned)v[0][1], (unsigned)v[1][1], false, false);
            if (prow >= 0) *reinterpret_cast<i32x4*>(dst + (32 * db + 16 * q) * 2) = i32x4{(int)s0[0], (int)s1[0], (int)s0[1], (int)s1[1]};
          }
      }
    }

    // ---- move on
    if (ticket(round + 1) >= ntickets) break;
    if constexpr (Tune::kEarlyQ) {
#pragma unroll
      for (int i = 0; i < KS; ++i) qreg[i] = nq[i];
    } else {
      load_q(qreg, nxt, tile_of(round + 1), a_seq);
    }
    my_scale = next_scale;
    my_blk = a_blk, seq = a_seq, a_blk = b_blk, a_seq = b_seq;
    cur = nxt, nxt = third, third = arrived(fourth);
  }
  FCA_WAIT_VMCNT(0);  // requests nobody uses are still in flight: let them land before the wave ends
}

hipError_t launch_attend_block_wide(const AttendParams& p, const fca_plan& plan, int cus, int max_workgroups, hipStream_t stream) {
  const MetaLayout L = make_layout(plan);
  const int64_t max_tickets = L.max_items * plan.num_kv_heads;
  int per_cu = WideTuning<64>::kWorkgroups;
  if (plan.head_dim == 256) per_cu = WideTuning<256>::kWorkgroups;
  int64_t grid = (int64_t)cus * per_cu;
  // The caller's cap leaves CUs to other streams, and a launch spreads over as many CUs as it has
  // workgroups: it counts them as they are, of two waves here.
  if (max_workgroups > 0 && max_workgroups < grid) grid = max_workgroups;
  if (grid > max_tickets) grid = max_tickets;
  if (grid < 1) grid = 1;
  // with sharing on, and but for query runs, a launch reads every KV block about once: past the caches
  const bool stream_kv = plan.max_levels > 0 && !p.kv_reread;
  hipEvent_t ev_start, ev_stop;
  take_attend_timing(&ev_start, &ev_stop);
#define FCA_LAUNCH(D_, S_) \
  if (ev_start) hipExtLaunchKernelGGL((fca_attend_block_wide_kernel<D_, S_>), dim3((unsigned)grid), dim3(128), 0, stream, ev_start, ev_stop, 0, p); \
  else hipLaunchKernelGGL((fca_attend_block_wide_kernel<D_, S_>), dim3((unsigned)grid), dim3(128), 0, stream, p)
#define FCA_PICK(D_) \
  if (stream_kv) { FCA_LAUNCH(D_, true); } else { FCA_LAUNCH(D_, false); }
  if (plan.head_dim == 256) {
    FCA_PICK(256);
  } else if (plan.head_dim == 128) {
    FCA_PICK(128);
  } else {
    FCA_PICK(64);
  }
#undef FCA_PICK
#undef FCA_LAUNCH
  return hipGetLastError();
}

}  // namespace fca
