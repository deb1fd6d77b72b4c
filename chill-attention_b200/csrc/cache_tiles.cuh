// Attention of MANY new tokens over a paged cache (trees, chunks of prompts), 16-bit types, on tcgen05: tiles of 128 rows (new
// tokens times the heads that share a kv head) and 64 keys.  See cache_common.cuh for units and shares.
//
// A CTA works on NQ tiles of rows of one kv head at once, which share the tiles of keys in its ring: with NQ = 2 keys go into shared
// memory once for 256 rows, and one tile's softmax runs beside the other one's products.
//   warps 0 .. 4 NQ - 1  softmax: thread r of a group owns row r of its tile: reads its row of S from TMEM, masks it where the tile of
//              keys needs it (one 64-bit word of visible keys: interval of the mask functor, ancestors of a tree, keys without a
//              page), follows the maximum lazily, writes P (16 bits) over S; in the end O / l or the piece's part
//   warp 4 NQ  producer: takes shares, hands their pieces to the other roles; Q by TMA (a tile begins at a token),
//              K and V in boxes of one page and 64 channels, a lane for each box; owns the TMEM allocation
//   next NQ warps  MMA issuer of each group (one for both took 3550 clocks for a step of two tiles, its instructions alone 2000: issuing a
//              product blocks for longer than it takes): S(j + 1) = Q K^T goes ahead of O += P(j) V, in two S buffers, so it
//              runs during the softmax of tile j
// TMEM columns of a group: two buffers of 64 for S / P, then O.
// Rounding as in the rows kernel: P once to 16 bits, sums of the unrounded weights in fp32.
#pragma once
#include "cache_common.cuh"
#include "cache_repair.cuh"
#include "tc_common.cuh"

#include <type_traits>

namespace chill {
namespace cache {

template <int DP, int NQ>
struct TilesShape {
  static_assert(NQ == 1 || DP <= 128, "TMEM holds one tile of head dim 256");
  static constexpr int kCtasPerSm = (DP <= 128 ? 2 : 1) / NQ;
  static constexpr int kChunks = DP / 64;
  static constexpr int kThreads = NQ == 1 ? 256 : 384;
  static constexpr int kGroupCols = 2 * kKeyTile + DP <= 128 ? 128 : (2 * kKeyTile + DP <= 256 ? 256 : 512);
  static constexpr int kTmemCols = NQ * kGroupCols;
  static constexpr int kQChunk = kTileRows * 128, kKvChunk = kKeyTile * 128;  // a 64-channel block
  static constexpr int kQTile = kTileRows * DP * 2;
  static constexpr int kKvBytes = kKeyTile * DP * 2;
  static constexpr int kStages = DP == 64 ? (NQ == 1 ? 5 : 8) : (NQ == 2 ? 5 : 2);
  static constexpr int kK = NQ * kQTile;
  static constexpr int kV = kK + kStages * kKvBytes;
  static constexpr int kBars = kV + kStages * kKvBytes;
  static constexpr int kNumBars = 3 * kStages + 6 + NQ * (3 * 2 + 2);
  static constexpr int kMisc = kBars + kNumBars * 8;
  static constexpr int kHoles = kMisc + 16;  // a word per stage
  static constexpr int kItems = (kHoles + kStages * 4 + 15) / 16 * 16;
  static constexpr int kCum = kItems + 2 * (int)sizeof(Item);
  static constexpr int kTotal = kCum + (kScanEntries + 1) * 4;
  static constexpr int kDynamic = kTotal + 1024;
  // a CTA's pool is threads x launch registers: NQ * softmax + other <= (NQ + 1) * launch
  static constexpr int kLaunchRegs = 65536 / (kCtasPerSm * kThreads) / 8 * 8 > 168 ? 168 : 65536 / (kCtasPerSm * kThreads) / 8 * 8;
  static constexpr int kSoftmaxRegs = NQ == 1 ? 184 : 208;
  static constexpr int kOtherRegs = NQ == 1 ? 72 : 88;
  static constexpr bool kSplit = DP <= 128;  // head dim 256: one CTA of 256 threads, every thread has enough
  static_assert(!kSplit || NQ * kSoftmaxRegs + kOtherRegs <= (NQ + 1) * kLaunchRegs, "setmaxnreg.inc would never be granted");
  static_assert(kCtasPerSm * (kDynamic + 1024) <= 233472 && kCtasPerSm * kTmemCols <= 512, "resources of an SM");
};

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3, int c4) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
               : "memory");
}

// 2^x of a pair on the FMA pipe: x = n + f, n = round(x) by adding 1.5 * 2^23, f in [-1/2, 1/2]; 2^f by a polynomial of degree 5 (minimax
// of the relative error by Remez' algorithm: 7.5e-8, evaluated in fp32 2.3e-7, as much as ex2.approx is off), n goes into the exponent.
__device__ __forceinline__ uint64_t ex2_fma(uint64_t x2) {
  float x0, x1;
  tc::upk2(x2, x0, x1);
  // below: 2^-126 beside a row's largest weight of 2^-8 or more; not for hidden keys, which need a 0, nor for scores that are not finite (NaN
  // becomes 2^-126 too): whoever calls this looks at the row's maximum
  x2 = tc::pk2(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t n2 = tc::fadd2(x2, tc::pk2(12582912.f, 12582912.f));
  const uint64_t f2 = tc::ffma2(tc::fadd2(n2, tc::pk2(-12582912.f, -12582912.f)), tc::pk2(-1.f, -1.f), x2);
  uint64_t p2 = tc::pk2(1.3276472e-3f, 1.3276472e-3f);
  p2 = tc::ffma2(p2, f2, tc::pk2(9.6755413e-3f, 9.6755413e-3f));
  p2 = tc::ffma2(p2, f2, tc::pk2(5.5507133e-2f, 5.5507133e-2f));
  p2 = tc::ffma2(p2, f2, tc::pk2(0.24022120f, 0.24022120f));
  p2 = tc::ffma2(p2, f2, tc::pk2(0.69314697f, 0.69314697f));
  p2 = tc::ffma2(p2, f2, tc::pk2(1.0000001f, 1.0000001f));
  float a, b, na, nb;
  tc::upk2(p2, a, b);
  tc::upk2(n2, na, nb);
  return tc::pk2u(__float_as_uint(a) + (__float_as_uint(na) << 23), __float_as_uint(b) + (__float_as_uint(nb) << 23));
}
// Of every sixteen pairs of weights, half as many are worked out so.  The two groups' softmax warps on a scheduler ask its MUFU for 1024
// of the 2100 clocks of a step, mostly at the same time: 1024 new tokens for each of 4 requests, 507 us with none, 480 with an eighth of
// the pairs, 467 with a quarter, 512 with half of them.
constexpr int kFmaShare = 8;

enum : int { kStTilesProducer = 711, kStTilesMma = 712, kStTilesSoftmax = 713, kStTilesEpilogue = 714 };

template <typename T, int DP, int NQ, class M>
__global__ void __launch_bounds__(TilesShape<DP, NQ>::kThreads, TilesShape<DP, NQ>::kCtasPerSm)
cached_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CachedP p) {
  using S = TilesShape<DP, NQ>;
  constexpr int kStages = S::kStages, kProducer = 4 * NQ;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - tc::smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // stages: k_full, v_full, free (O += P V of every group is done, K and V may be replaced); items: item_full, item_empty, q_full, q_empty
  const uint32_t k_full = base + S::kBars, v_full = k_full + 8 * kStages, kv_free = v_full + 8 * kStages, item_full = kv_free + 8 * kStages,
                 item_empty = item_full + 16, q_full = item_empty + 16, q_empty = q_full + 8;
  // of group g, + g * 64: s_full[2], p_full[2], pv_done[2], o_full, o_empty
  const uint32_t group_bars = q_empty + 8;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + S::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + S::kMisc + 4);
  volatile int* holes = reinterpret_cast<volatile int*>(gen + S::kHoles);
  Item* items = reinterpret_cast<Item*>(gen + S::kItems);
  const tc::Guard guard{p.status, abort_flag};
  if (threadIdx.x == 0) {
    abort_flag[0] = 0;
    abort_flag[1] = kFirstLimit;
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(k_full + 8 * s, 1);
      tc::mbar_init(v_full + 8 * s, 1);
      tc::mbar_init(kv_free + 8 * s, NQ);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(item_full + 8 * s, 1);
      tc::mbar_init(item_empty + 8 * s, 5 * NQ);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, NQ);
    for (int g = 0; g < NQ; ++g) {
      for (int s = 0; s < 2; ++s) {
        tc::mbar_init(group_bars + 64 * g + 8 * s, 1);
        tc::mbar_init(group_bars + 64 * g + 16 + 8 * s, 4);
        tc::mbar_init(group_bars + 64 * g + 32 + 8 * s, 1);
      }
      tc::mbar_init(group_bars + 64 * g + 48, 1);
      tc::mbar_init(group_bars + 64 * g + 56, 4);
    }
    tc::fence_barrier_init();
  }
  // rows of Q behind the last whole token are never loaded
  for (int idx = threadIdx.x; idx < NQ * S::kQTile / 16; idx += S::kThreads) *reinterpret_cast<uint4*>(gen + idx * 16) = make_uint4(0u, 0u, 0u, 0u);
  tc::fence_proxy_async_smem();
  if (warp == kProducer) {
    tc::tmem_alloc(tc::smem_u32(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
    tc::tmem_relinquish();
  }
  const int* cum;
  const Cut cut = begin_work<M, S::kThreads>(p, reinterpret_cast<int*>(gen + S::kCum), cum);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();

  if (warp == kProducer) {
    if constexpr (S::kSplit) tc::reg_dealloc<S::kOtherRegs>();
    // ---------------------------------------------------------------------------------------------- producer
    const int boxes = kKeyTile / p.box, jobs = boxes * S::kChunks, mine = lane % boxes;
    const uint32_t box_bytes = (uint32_t)p.box * 128u;
    const int half = p.rows / NQ, tokens = half / p.G;  // rows and tokens of one group's tile
    int n = 0, loads = 0;
    bool ok = true;
    Work work;
    work.start<M>(p, cut, cum);
    Item it;
    for (int item = 0;; ++item) {
      const bool more = work.next<M>(p, it);
      const int slot = item & 1;
      ok = __all_sync(0xffffffffu, bounded_wait(item_empty + 8 * slot, ((uint32_t)(item >> 1) & 1u) ^ 1u, guard, kStTilesProducer));
      if (!ok) break;
      const RowTile& t = it.t;
      if (lane == 0) {
        items[slot] = it;
        tc::mbar_arrive(item_full + 8 * slot);
      }
      __syncwarp();
      if (!more) break;
      if (it.x.t0 >= it.tiles) continue;
      bool there = false, there_next = false;
      int page = 0, page_next = tile_page(p, t, t.k_lo + it.x.t0 * kKeyTile, mine, there_next);
      // Q: the last product with the piece before's is done
      ok = __all_sync(0xffffffffu, bounded_wait(q_empty, ((uint32_t)loads & 1u) ^ 1u, guard, kStTilesProducer));
      if (!ok) break;
      ++loads;
      if (lane == 0) tc::mbar_arrive_expect_tx(q_full, (uint32_t)(NQ * half * S::kChunks * 128));
      __syncwarp();
      if (lane < NQ * S::kChunks) {
        const int g = lane / S::kChunks, c = lane % S::kChunks;
        tma_load_5d(base + g * S::kQTile + c * S::kQChunk, &tmQ, q_full, c * 64, 0, (t.r0 + g * half) / p.G, it.x.head, t.b);
      }
      for (int kt = it.x.t0; kt < it.tiles; ++kt, ++n) {
        const int s = n % kStages, k0 = t.k_lo + kt * kKeyTile, row = (k0 + mine * p.box) % p.page;
        page = page_next;
        there = there_next;
        if (kt + 1 < it.tiles) page_next = tile_page(p, t, k0 + kKeyTile, mine, there_next);
        const unsigned lost = __ballot_sync(0xffffffffu, !there && lane < boxes);
        ok = __all_sync(0xffffffffu, bounded_wait(kv_free + 8 * s, ((uint32_t)(n / kStages) & 1u) ^ 1u, guard, kStTilesProducer));
        if (!ok) break;
        if (lane == 0) {
          holes[s] = lost_groups(p, lost, boxes);
          tc::mbar_arrive_expect_tx(k_full + 8 * s, S::kKvBytes);
          tc::mbar_arrive_expect_tx(v_full + 8 * s, S::kKvBytes);
        }
        __syncwarp();
        for (int j = lane; j < jobs; j += 32)
          tc::tma_load_4d(base + S::kK + s * S::kKvBytes + (j / boxes) * S::kKvChunk + mine * box_bytes, &tmK, k_full + 8 * s, (j / boxes) * 64, row, it.x.head, page);
        for (int j = lane; j < jobs; j += 32)
          tc::tma_load_4d(base + S::kV + s * S::kKvBytes + (j / boxes) * S::kKvChunk + mine * box_bytes, &tmV, v_full + 8 * s, (j / boxes) * 64, row, it.x.head, page);
      }
      if (!ok) break;
    }
    if (!ok) {  // copies already in flight land before the CTA's shared memory goes away
      const uint64_t t0 = tc::globaltimer_ns();
      while (tc::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
  } else if (warp <= kProducer + NQ && warp > kProducer) {
    if constexpr (S::kSplit) tc::reg_dealloc<S::kOtherRegs>();
    // -------------------------------------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = tc::make_idesc<T>(kTileRows, kKeyTile, false, false);
    constexpr uint32_t idesc_o = tc::make_idesc<T>(kTileRows, DP, false, true);
    constexpr uint32_t hi = tc::desc_hi_sw128(1024);  // both operand kinds: 8-row groups 1 KB apart
    const uint32_t g = (uint32_t)(warp - kProducer - 1), cols = tmem + g * S::kGroupCols;
    const uint32_t s_full = group_bars + 64 * g, p_full = s_full + 16, pv_done = s_full + 32, o_full = s_full + 48, o_empty = s_full + 56;
    const uint32_t q_lo = tc::desc_lo_sw128(base + g * S::kQTile, 16);
    int pieces = 0;
    // tile x: its stage (slot and phase) for S and for O += P V, counted along
    int s_slot = 0, v_slot = 0;
    uint32_t s_phase = 0, v_phase = 0, n = 0;
    bool ok = true;
    for (int item = 0; ok; ++item) {
      const int slot = item & 1;
      ok = __all_sync(0xffffffffu, bounded_wait(item_full + 8 * slot, (uint32_t)(item >> 1) & 1u, guard, kStTilesMma));
      if (!ok) break;
      const int entry = items[slot].x.entry, count = items[slot].tiles - items[slot].x.t0;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(item_empty + 8 * slot);
      if (entry < 0) break;
      if (count <= 0) continue;
      if (lane == 0) {
        auto issue_s = [&](uint32_t sb) -> bool {  // S = Q K^T; the buffer's P has been used by a product issued before
          const uint32_t k_lo = tc::desc_lo_sw128(base + S::kK + s_slot * S::kKvBytes, 16);
          if (!bounded_wait(k_full + 8 * s_slot, s_phase, guard, kStTilesMma)) return false;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            tc::mma_ss_lh(cols + sb * kKeyTile, q_lo + tc::kmajor_step(kk), k_lo + (uint32_t)((kk / 4) * (S::kKvChunk / 16) + (kk % 4) * 2), hi, idesc_s, kk > 0 ? 1u : 0u);
          tc::mma_commit(s_full + 8 * sb);
          if (++s_slot == kStages) s_slot = 0, s_phase ^= 1u;
          return true;
        };
        ok = bounded_wait(q_full, (uint32_t)pieces & 1u, guard, kStTilesMma);
        if (ok) ok = issue_s(n & 1u);
        for (int j = 0; j < count && ok; ++j, ++n) {
          if (j + 1 < count) ok = issue_s((n + 1) & 1u);
          if (!ok) break;
          const bool first = j == 0;
          const uint32_t sb = n & 1u, v_lo = tc::desc_lo_sw128(base + S::kV + v_slot * S::kKvBytes, S::kKvChunk);  // MN-major: channel blocks one chunk apart
          if (!(ok = bounded_wait(v_full + 8 * v_slot, v_phase, guard, kStTilesMma))) break;
          if (first && !(ok = bounded_wait(o_empty, ((uint32_t)pieces & 1u) ^ 1u, guard, kStTilesMma))) break;
          if (!(ok = bounded_wait(p_full + 8 * sb, (n >> 1) & 1u, guard, kStTilesMma))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kKeyTile / 16; ++kk)  // O += P V
            tc::mma_ts_lh(cols + 2 * kKeyTile, cols + sb * kKeyTile + kk * 8, v_lo + kk * 128, hi, idesc_o, (!first || kk > 0) ? 1u : 0u);
          tc::mma_commit(kv_free + 8 * v_slot);
          if (NQ > 1) tc::mma_commit(pv_done + 8 * sb);
          if (++v_slot == kStages) v_slot = 0, v_phase ^= 1u;
        }
        if (ok) {
          tc::mma_commit(o_full);
          tc::mma_commit(q_empty);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      ++pieces;
    }
  } else if (warp > kProducer + NQ) {
    if constexpr (S::kSplit) tc::reg_dealloc<S::kOtherRegs>();
  } else {
    if constexpr (S::kSplit) tc::reg_alloc<S::kSoftmaxRegs>();
    // ------------------------------------------------------------------------------------ softmax and epilogue
    const int grp = NQ == 1 ? 0 : warp >> 2, r = (warp & 3) * 32 + lane;  // row of the group's tile == TMEM lane
    const uint32_t lane_sel = ((uint32_t)((warp & 3) * 32) << 16) + grp * S::kGroupCols;
    const uint32_t s_full = group_bars + 64 * grp, p_full = s_full + 16, o_full = s_full + 48, o_empty = s_full + 56;
    const uint32_t tO = tmem + 2 * kKeyTile + lane_sel;
    const float c = p.scale_log2;
    const int half = p.rows / NQ;
    int n = 0, pieces = 0;
    for (int item = 0;; ++item) {
      const int slot = item & 1;
      // The warps leave together: whether there is one more piece, and whether all of them saw it, is settled at a barrier
      bool leave = !__all_sync(0xffffffffu, bounded_wait(item_full + 8 * slot, (uint32_t)(item >> 1) & 1u, guard, kStTilesSoftmax));
      if (!leave) leave = items[slot].x.entry < 0;
      if (consumers_any(leave, 2 + grp)) break;
      const RowTile& t = items[slot].t;
      const Piece& piece = items[slot].x;
      const int t0 = piece.t0, count = imax(items[slot].tiles - t0, 0), k_lo = t.k_lo, total = t.total, full_lo = t.full_lo, full_hi = t.full_hi;
      const int row = grp * half + r;  // of the unit
      const int i = r < half && row < t.rows ? (t.r0 + row) / p.G : -1;
      const int pos = i >= 0 ? token_position(p, t, i) : 0;
      const uint64_t near = first_ancestors(p, t.b, i);
      float m_used = -CUDART_INF_F, l = 0.f;
      bool ok = true;
      for (int j = 0; j < count; ++j, ++n) {
        const int s = n % kStages, sb = n & 1, k0 = k_lo + (t0 + j) * kKeyTile;
        const uint32_t tS = tmem + sb * kKeyTile + lane_sel;
        ok = __all_sync(0xffffffffu, bounded_wait(s_full + 8 * sb, (uint32_t)(n >> 1) & 1u, guard, kStTilesSoftmax));
        if (!ok) break;
        tc::tc_fence_after();
        const int lost = holes[s];
        const bool full = lost == 0 && k0 >= full_lo && k0 + kKeyTile <= full_hi;
        uint64_t vis = ~0ull;
        if (!full) vis = visible_keys<M>(p, t, i, pos, near, k0, lost);
        __syncwarp();
        uint32_t x[kKeyTile];
        tc::tmem_ld32(tS, x);
        tc::tmem_ld32(tS + 32, x + 32);
        tc::tmem_wait_ld();
        if (!full) {
          const uint32_t lo = (uint32_t)vis, hi = (uint32_t)(vis >> 32);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            x[e] = (lo >> e) & 1u ? x[e] : 0xff800000u;
            x[32 + e] = (hi >> e) & 1u ? x[32 + e] : 0xff800000u;
          }
        }
        float mx0 = -CUDART_INF_F, mx1 = mx0, mx2 = mx0, mx3 = mx0;
#pragma unroll
        for (int e = 0; e < kKeyTile; e += 8) {
          mx0 = tc::fmax3_nan(mx0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
          mx1 = tc::fmax3_nan(mx1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          mx2 = tc::fmax3_nan(mx2, __uint_as_float(x[e + 4]), __uint_as_float(x[e + 5]));
          mx3 = tc::fmax3_nan(mx3, __uint_as_float(x[e + 6]), __uint_as_float(x[e + 7]));
        }
        const float top = tc::fmax3_nan(tc::fmax3_nan(mx0, mx1, mx2), mx3, mx3);
        const float m_cand = fmaxf(m_used, top * c);  // passes NaN by
        if (j == 0) {
          m_used = m_cand;
        } else if (__any_sync(0xffffffffu, m_cand - m_used > 8.f)) {  // lazily: O is rescaled when the maximum grew by more than 2^8
          // the accumulation of the tile before must be done before O is touched
          const uint32_t done = NQ == 1 ? kv_free + 8 * (uint32_t)((n - 1) % kStages) : s_full + 32 + 8 * (uint32_t)((n - 1) & 1);
          const uint32_t parity = (uint32_t)((n - 1) / (NQ == 1 ? kStages : 2)) & 1u;
          ok = __all_sync(0xffffffffu, bounded_wait(done, parity, guard, kStTilesSoftmax));
          if (!ok) break;
          tc::tc_fence_after();
          const bool moves = m_cand - m_used > 8.f;  // a row goes by itself: rows that do not exist hold anything
          const float a = moves ? tc::ex2(m_used - m_cand) : 1.f;
          l *= a;
          m_used = moves ? m_cand : m_used;
#pragma unroll 1
          for (int d = 0; d < DP; d += 16) {
            uint32_t o[16];
            tc::tmem_ld16(tO + d, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tc::tmem_st16(tO + d, o);
          }
        }
        const float safe = m_used == -CUDART_INF_F ? 0.f : m_used;
        const uint64_t c2 = tc::pk2(c, c), nm2 = tc::pk2(-safe, -safe);
        uint64_t l0 = 0ull, l1 = 0ull;
        auto weights = [&](auto fma) {
#pragma unroll
          for (int e = 0; e < kKeyTile / 2; e += 2) {
            const uint64_t a0 = tc::ffma2(tc::pk2u(x[2 * e], x[2 * e + 1]), c2, nm2), a1 = tc::ffma2(tc::pk2u(x[2 * e + 2], x[2 * e + 3]), c2, nm2);
            const uint64_t e0 = decltype(fma)::value && e % 16 < kFmaShare ? ex2_fma(a0) : tc::ex2_pair(a0, false);
            const uint64_t e1 = tc::ex2_pair(a1, false);
            l0 = tc::fadd2(l0, e0);
            l1 = tc::fadd2(l1, e1);
            float p0, p1, p2, p3;
            tc::upk2(e0, p0, p1);
            tc::upk2(e1, p2, p3);
            x[e] = tc::pack2<T>(p0, p1);  // a slot that has been used already (e <= 2 e)
            x[e + 1] = tc::pack2<T>(p2, p3);
          }
        };
        if (full) weights(std::true_type{});
        else weights(std::false_type{});
        float a0, a1, a2, a3;
        tc::upk2(l0, a0, a1);
        tc::upk2(l1, a2, a3);
        l += (a0 + a1) + (a2 + a3);
        // The weights on the FMA pipe know neither NaN nor infinity.  A score of NaN or +inf, or nothing but -inf, shows in the tile's maximum:
        // 0 times that is NaN, and the sum that holds it sends the piece to repair_piece
        if (full) l = fmaf(top, 0.f, l);
        tc::tmem_st32(tS, x);
        if (k0 + kKeyTile > total) {  // rows of V behind the last key may hold anything, and 0 * NaN is NaN: they become 0
          ok = __all_sync(0xffffffffu, bounded_wait(v_full + 8 * s, (uint32_t)(n / kStages) & 1u, guard, kStTilesSoftmax));
          if (!ok) break;
          const int gone = imax(total - k0, 0);
          // both groups write the same zeros: neither's product may start before its own have been written
          for (int idx = r; idx < (kKeyTile - gone) * (DP / 8); idx += 128) {
            const int key = gone + idx / (DP / 8), u = idx % (DP / 8);
            *reinterpret_cast<uint4*>(gen + S::kV + s * S::kKvBytes + (u / 8) * S::kKvChunk + key * 128 + (u % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          tc::fence_proxy_async_smem();
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full + 8 * sb);
      }
      if (ok && count > 0) ok = __all_sync(0xffffffffu, bounded_wait(o_full, (uint32_t)pieces & 1u, guard, kStTilesEpilogue));
      tc::tc_fence_after();
      const int unit_row = t.r0 + row;
      const bool exists = r < half && unit_row < p.N * p.G;
      const int out_i = unit_row / p.G, out_h = piece.head * p.G + unit_row % p.G;
      bool odd = i >= 0 && !(l <= 3e38f);
      const float inv = i >= 0 && l != 0.f ? 1.f / l : 0.f;
      T* to = o_row<T>(p, t.b, out_h, out_i);
      float4* part = reinterpret_cast<float4*>(p.part_o) + (long long)imax(piece.slot, 0) * (p.D / 4) * p.rows + row;  // [D / 4][row]: lanes side by side
#pragma unroll 1
      for (int d = 0; d < DP; d += 32) {
        uint32_t o[32];
        __syncwarp();
        if (count > 0 && ok) {
          tc::tmem_ld32(tO + d, o);
          tc::tmem_wait_ld();
        }
        if (count == 0 || !ok || i < 0) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!exists || d >= p.D) continue;
        float big = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) big += fabsf(__uint_as_float(o[e]));
        odd |= i >= 0 && !(big <= 3e38f);
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (d + e >= p.D) break;
          float f[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) f[u] = __uint_as_float(o[e + u]);
          if (piece.slot >= 0) {
            part[(long long)((d + e) / 4) * p.rows] = make_float4(f[0], f[1], f[2], f[3]);
            part[(long long)((d + e) / 4 + 1) * p.rows] = make_float4(f[4], f[5], f[6], f[7]);
          } else if (p.wide_o) {
            *reinterpret_cast<uint4*>(to + d + e) = make_uint4(tc::pack2<T>(f[0] * inv, f[1] * inv), tc::pack2<T>(f[2] * inv, f[3] * inv),
                                                               tc::pack2<T>(f[4] * inv, f[5] * inv), tc::pack2<T>(f[6] * inv, f[7] * inv));
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u) to[(d + e + u) * p.o.sd] = from_f<T>(f[u] * inv);
          }
        }
      }
      if (exists) {
        if (piece.slot < 0) store_lse(p, t.b, out_h, out_i, i >= 0, m_used, l);
        else p.part_ml[(long long)piece.slot * p.rows + row] = make_float2(m_used, l);
      }
      if (count > 0) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(o_empty);
        ++pieces;
      }
      if (consumers_any(odd, 2 + grp)) repair_piece<T, DP, M, true>(p, t, piece, grp * half + (warp & 3), 4, (grp + 1) * half, abort_flag + 1);
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(item_empty + 8 * slot);
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == kProducer) tc::tmem_dealloc(tmem, S::kTmemCols);
}

}  // namespace cache
}  // namespace chill
