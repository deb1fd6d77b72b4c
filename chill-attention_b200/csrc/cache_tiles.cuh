// Attention of MANY new tokens over a paged cache (trees, chunks of prompts), 16-bit types, on tcgen05: tiles of 128 rows (new
// tokens times the heads that share a kv head) and 64 keys.  See cache_common.cuh for units and shares.
//
// The CTAs are persistent (two on an SM up to head dim 128, one at 256) and walk their shares piece by piece:
//   warps 0-3  softmax: thread r owns row r; writes its row of Q into shared memory (rows of a tile are token-major, a gather for
//              any number of heads in a group), per tile reads its row of S from TMEM, masks it where the tile needs it (one 64-bit
//              word of visible keys per row: interval of the mask functor, ancestors of a tree, keys without a page), follows the
//              maximum lazily, writes P (16 bits) over S; in the end O / l or the piece's part
//   warp 4     producer: boxes of one page and 64 channels by TMA, a lane for each box; owns the TMEM allocation
//   warp 5     MMA issuer: S(j + 1) = Q K^T goes ahead of O += P(j) V, in two S buffers, so it runs during the softmax of tile j
// TMEM columns: two buffers of 64 for S / P, then O.
// Rounding as in the rows kernel: P once to 16 bits, sums of the unrounded weights in fp32.
#pragma once
#include "cache_common.cuh"
#include "cache_repair.cuh"
#include "tc_common.cuh"

namespace chill {
namespace cache {

constexpr int kTileRows = 128;
constexpr int kTilesThreads = 256;

template <int DP>
struct TilesShape {
  static constexpr int kCtasPerSm = DP <= 128 ? 2 : 1;
  static constexpr int kChunks = DP / 64;
  static constexpr int kStages = 2;
  static constexpr int kTmemCols = 2 * kKeyTile + DP <= 256 ? 256 : 512;
  static constexpr int kQChunk = kTileRows * 128, kKvChunk = kKeyTile * 128;  // a 64-channel block
  static constexpr int kKvBytes = kKeyTile * DP * 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kTileRows * DP * 2;
  static constexpr int kV = kK + kStages * kKvBytes;
  static constexpr int kBars = kV + kStages * kKvBytes;
  static constexpr int kMisc = kBars + 16 * 8;
  static constexpr int kHoles = kMisc + 16;  // four words: the producer may be two tiles ahead of the softmax of a stage
  static constexpr int kCum = kHoles + 16;
  static constexpr int kTotal = kCum + (kScanEntries + 4) * 4;
  static constexpr int kDynamic = kTotal + 1024;
  static constexpr int kSoftmaxRegs = 200, kOtherRegs = 56;  // two CTAs on an SM: 2 * 128 * (200 + 56) = 65536
  static_assert(kCtasPerSm * (kDynamic + 1024) <= 233472 && kCtasPerSm * kTmemCols <= 512, "resources of an SM");
};

enum : int { kStTilesProducer = 711, kStTilesMma = 712, kStTilesSoftmax = 713, kStTilesEpilogue = 714 };

// Keys k0 .. k0 + 63 that a row sees (token i at position pos), as bits.
template <class M>
__device__ __forceinline__ uint64_t visible_keys(const CachedP& p, const RowTile& t, int i, int pos, int k0, int lost) {
  const int n = t.cached + t.fresh, there = imin(t.total - k0, kKeyTile);
  if (i < 0 || there <= 0) return 0ull;
  const bool tree = p.ancestors != nullptr;
  auto below = [](int c) -> uint64_t { return c >= 64 ? ~0ull : (c <= 0 ? 0ull : (1ull << c) - 1ull); };
  // by the mask functor: all keys of a chain, the cached ones of a tree
  const int cols = tree ? imin(t.cached - k0, there) : there;
  uint64_t vis = 0ull;
  if (cols > 0) {
    if (interval_rows<M>::value) {
      int lo, hi;
      row_window<M, true>(pos, k0, cols, n, p.margs, lo, hi);
      vis = below(hi + 1) & ~below(lo);
    } else {
      for (int c = 0; c < cols; ++c)
        if (M::mask(pos, k0 + c, n, p.margs)) vis |= 1ull << c;
    }
  }
  if (tree && k0 + there > t.cached) {  // by ancestry, then by the mask at the ancestors' positions
    const int* row = p.ancestors + ((long long)t.b * p.N + i) * p.words;
    const int j0 = k0 - t.cached;  // number of the new token at the tile's first key
    const int w = imax(j0, 0) >> 5, sh = imax(j0, 0) & 31;
    auto word = [&](int x) -> uint64_t { return x < p.words ? (uint64_t)(unsigned)row[x] : 0ull; };
    uint64_t bits = (word(w) | (word(w + 1) << 32)) >> sh;
    if (sh != 0) bits |= word(w + 2) << (64 - sh);
    if (j0 < 0) bits <<= -j0;
    bits &= below(there);
    const int* at = p.positions + (long long)t.b * p.N + j0;
    for (uint64_t left = bits; left != 0ull;) {
      const int c = __ffsll((long long)left) - 1;
      left &= left - 1ull;
      if (!M::mask(pos, at[c], n, p.margs)) bits &= ~(1ull << c);
    }
    vis |= bits;
  }
  for (int g = lost; g != 0; g &= g - 1) vis &= ~(0xffull << (8 * (__ffs(g) - 1)));
  return vis;
}

template <typename T, int DP, class M>
__global__ void __launch_bounds__(kTilesThreads, TilesShape<DP>::kCtasPerSm)
cached_tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CachedP p) {
  using S = TilesShape<DP>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - tc::smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bars = base + S::kBars;
  // s_full[s]: S(n) is there and K stage s = n % 2 is free; v_empty[s]: O += P(n) V is done, V stage s is free
  const uint32_t k_full = bars, v_full = bars + 16, s_full = bars + 32, v_empty = bars + 48, p_full = bars + 64, q_full = bars + 80, o_full = bars + 88,
                 o_empty = bars + 96;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + S::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + S::kMisc + 4);
  volatile int* holes = reinterpret_cast<volatile int*>(gen + S::kHoles);
  const tc::Guard guard{p.status, abort_flag};
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(k_full + 8 * s, 1);
      tc::mbar_init(v_full + 8 * s, 1);
      tc::mbar_init(s_full + 8 * s, 1);
      tc::mbar_init(v_empty + 8 * s, 1);
      tc::mbar_init(p_full + 8 * s, 4);
    }
    tc::mbar_init(q_full, 4);
    tc::mbar_init(o_full, 1);
    tc::mbar_init(o_empty, 4);
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
  }
  if (warp == 4) {
    tc::tmem_alloc(tc::smem_u32(const_cast<uint32_t*>(tmem_slot)), S::kTmemCols);
    tc::tmem_relinquish();
  }
  const int* cum;
  Share share = begin_share<M, kTilesThreads>(p, reinterpret_cast<int*>(gen + S::kCum), cum);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = *tmem_slot, tO = tmem + 2 * kKeyTile;
  Piece piece;

  if (warp == 4) {
    if constexpr (S::kCtasPerSm > 1) tc::reg_dealloc<S::kOtherRegs>();
    // ---------------------------------------------------------------------------------------------- producer
    const int boxes = kKeyTile / p.box, jobs = boxes * S::kChunks, mine = lane % boxes;
    const uint32_t box_bytes = (uint32_t)p.box * 128u;
    int n = 0;
    bool ok = true;
    while (ok && share.next(p, cum, piece)) {
      const RowTile t = row_tile<M>(p, piece.entry);
      const int tiles = t.n_tiles == 0 ? 0 : piece.t1;
      bool there = false, there_next = false;
      int page = 0, page_next = 0;
      if (piece.t0 < tiles) page_next = tile_page(p, t, t.k_lo + piece.t0 * kKeyTile, mine, there_next);
      for (int kt = piece.t0; kt < tiles; ++kt, ++n) {
        const int s = n & 1, k0 = t.k_lo + kt * kKeyTile, row = (k0 + mine * p.box) % p.page;
        const uint32_t again = ((uint32_t)(n >> 1) & 1u) ^ 1u;
        page = page_next;
        there = there_next;
        if (kt + 1 < tiles) page_next = tile_page(p, t, k0 + kKeyTile, mine, there_next);
        const unsigned lost = __ballot_sync(0xffffffffu, !there && lane < boxes);
        ok = __all_sync(0xffffffffu, tc::mbar_wait(s_full + 8 * s, again, guard, kStTilesProducer));
        if (!ok) break;
        if (lane == 0) {
          holes[n & 3] = lost_groups(p, lost, boxes);
          tc::mbar_arrive_expect_tx(k_full + 8 * s, S::kKvBytes);
        }
        __syncwarp();
        for (int j = lane; j < jobs; j += 32)
          tc::tma_load_4d(base + S::kK + s * S::kKvBytes + (j / boxes) * S::kKvChunk + mine * box_bytes, &tmK, k_full + 8 * s, (j / boxes) * 64, row, piece.head, page);
        ok = __all_sync(0xffffffffu, tc::mbar_wait(v_empty + 8 * s, again, guard, kStTilesProducer));
        if (!ok) break;
        if (lane == 0) tc::mbar_arrive_expect_tx(v_full + 8 * s, S::kKvBytes);
        __syncwarp();
        for (int j = lane; j < jobs; j += 32)
          tc::tma_load_4d(base + S::kV + s * S::kKvBytes + (j / boxes) * S::kKvChunk + mine * box_bytes, &tmV, v_full + 8 * s, (j / boxes) * 64, row, piece.head, page);
      }
    }
    if (!ok) {  // copies already in flight land before the CTA's shared memory goes away
      const uint64_t t0 = tc::globaltimer_ns();
      while (tc::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
  } else if (warp == 5) {
    if constexpr (S::kCtasPerSm > 1) tc::reg_dealloc<S::kOtherRegs>();
    // -------------------------------------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = tc::make_idesc<T>(kTileRows, kKeyTile, false, false);
    constexpr uint32_t idesc_o = tc::make_idesc<T>(kTileRows, DP, false, true);
    constexpr uint32_t hi = tc::desc_hi_sw128(1024);  // both operand kinds: 8-row groups 1 KB apart
    const uint32_t q_lo = tc::desc_lo_sw128(base + S::kQ, 16);
    int n = 0, pieces = 0;
    bool ok = true;
    while (ok && share.next(p, cum, piece)) {
      const RowTile t = row_tile<M>(p, piece.entry);
      const int tiles = t.n_tiles == 0 ? 0 : piece.t1, count = tiles - piece.t0;
      if (count <= 0) continue;
      if (lane == 0) {
        auto issue_s = [&](int x) -> bool {  // S(x) = Q K(x)^T
          const int s = x & 1;
          if (!tc::mbar_wait(k_full + 8 * s, (uint32_t)(x >> 1) & 1u, guard, kStTilesMma)) return false;
          tc::tc_fence_after();
          const uint32_t k_lo = tc::desc_lo_sw128(base + S::kK + s * S::kKvBytes, 16);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            tc::mma_ss_lh(tmem + s * kKeyTile, q_lo + tc::kmajor_step(kk), k_lo + (uint32_t)((kk / 4) * (S::kKvChunk / 16) + (kk % 4) * 2), hi, idesc_s, kk > 0 ? 1u : 0u);
          tc::mma_commit(s_full + 8 * s);
          return true;
        };
        auto issue_pv = [&](int x, bool first) -> bool {  // O += P(x) V(x)
          const int s = x & 1;
          if (!tc::mbar_wait(p_full + 8 * s, (uint32_t)(x >> 1) & 1u, guard, kStTilesMma)) return false;
          if (!tc::mbar_wait(v_full + 8 * s, (uint32_t)(x >> 1) & 1u, guard, kStTilesMma)) return false;
          if (first && !tc::mbar_wait(o_empty, ((uint32_t)pieces & 1u) ^ 1u, guard, kStTilesMma)) return false;
          tc::tc_fence_after();
          const uint32_t v_lo = tc::desc_lo_sw128(base + S::kV + s * S::kKvBytes, S::kKvChunk);  // MN-major: channel blocks one chunk apart
#pragma unroll
          for (int kk = 0; kk < kKeyTile / 16; ++kk)
            tc::mma_ts_lh(tO, tmem + s * kKeyTile + kk * 8, v_lo + kk * 128, hi, idesc_o, (!first || kk > 0) ? 1u : 0u);
          tc::mma_commit(v_empty + 8 * s);
          return true;
        };
        ok = tc::mbar_wait(q_full, (uint32_t)pieces & 1u, guard, kStTilesMma);
        tc::tc_fence_after();
        if (ok) ok = issue_s(n);
        for (int j = 0; j < count && ok; ++j) {
          if (j + 1 < count) ok = issue_s(n + j + 1);
          if (ok) ok = issue_pv(n + j, j == 0);
        }
        if (ok) tc::mma_commit(o_full);
      }
      ok = __all_sync(0xffffffffu, ok);
      n += count;
      ++pieces;
    }
  } else if (warp > 5) {
    if constexpr (S::kCtasPerSm > 1) tc::reg_dealloc<S::kOtherRegs>();
  } else {
    if constexpr (S::kCtasPerSm > 1) tc::reg_alloc<S::kSoftmaxRegs>();
    // ------------------------------------------------------------------------------------ softmax and epilogue
    const int r = warp * 32 + lane;
    const uint32_t lane_sel = (uint32_t)(warp * 32) << 16;
    const float c = p.scale_log2;
    int n = 0, pieces = 0;
    while (share.next(p, cum, piece)) {  // after a wait that ran out, too: all warps meet at the pieces' barriers
      const RowTile t = row_tile<M>(p, piece.entry);
      const int tiles = t.n_tiles == 0 ? 0 : piece.t1, count = imax(tiles - piece.t0, 0);
      const int i = r < t.rows ? (t.r0 + r) / p.G : -1;
      const bool exists = t.r0 + r < p.N * p.G;
      const int out_i = (t.r0 + r) / p.G, out_h = piece.head * p.G + (t.r0 + r) % p.G;
      const int pos = i >= 0 ? token_position(p, t, i) : 0;
      float m_used = -CUDART_INF_F, l = 0.f;
      bool ok = true;
      if (count > 0) {
        // Q: the MMAs of the piece before are complete (this thread has seen its last S)
        const T* src = row_ptr<T>(p.q, t.b, out_h, out_i);
#pragma unroll 4
        for (int u = 0; u < DP / 8; ++u) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (i >= 0 && u * 8 < p.D) {
            if (p.wide_q) {
              x = *reinterpret_cast<const uint4*>(src + u * 8);
            } else {
              T e[8];
#pragma unroll
              for (int v = 0; v < 8; ++v) e[v] = src[(u * 8 + v) * p.q.sd];
              x = *reinterpret_cast<const uint4*>(e);
            }
          }
          *reinterpret_cast<uint4*>(gen + S::kQ + (u / 8) * S::kQChunk + r * 128 + (((u % 8) ^ (r & 7)) * 16)) = x;
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(q_full);
      }
      for (int j = 0; j < count; ++j, ++n) {
        const int s = n & 1, k0 = t.k_lo + (piece.t0 + j) * kKeyTile;
        const uint32_t tS = tmem + s * kKeyTile + lane_sel, parity = (uint32_t)(n >> 1) & 1u;
        ok = __all_sync(0xffffffffu, tc::mbar_wait(s_full + 8 * s, parity, guard, kStTilesSoftmax));
        if (!ok) break;
        tc::tc_fence_after();
        const int lost = holes[n & 3];
        const bool full = lost == 0 && k0 >= t.full_lo && k0 + kKeyTile <= t.full_hi;
        uint64_t vis = ~0ull;
        if (!full) vis = visible_keys<M>(p, t, i, pos, k0, lost);
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
          mx0 = tc::fmax3(mx0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
          mx1 = tc::fmax3(mx1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          mx2 = tc::fmax3(mx2, __uint_as_float(x[e + 4]), __uint_as_float(x[e + 5]));
          mx3 = tc::fmax3(mx3, __uint_as_float(x[e + 6]), __uint_as_float(x[e + 7]));
        }
        const float m_cand = fmaxf(m_used, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * c);
        if (j == 0) {
          m_used = m_cand;
        } else if (__any_sync(0xffffffffu, m_cand - m_used > 8.f)) {  // lazily: O is rescaled when the maximum grew by more than 2^8
          // the accumulation of the tile before must be done before O is touched
          ok = __all_sync(0xffffffffu, tc::mbar_wait(v_empty + 8 * (uint32_t)((n - 1) & 1), (uint32_t)((n - 1) >> 1) & 1u, guard, kStTilesSoftmax));
          if (!ok) break;
          tc::tc_fence_after();
          const float a = m_cand == -CUDART_INF_F ? 1.f : tc::ex2(m_used - m_cand);
          l *= a;
          m_used = m_cand;
#pragma unroll 1
          for (int d = 0; d < DP; d += 16) {
            uint32_t o[16];
            tc::tmem_ld16(tO + lane_sel + d, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tc::tmem_st16(tO + lane_sel + d, o);
          }
        }
        const float safe = m_used == -CUDART_INF_F ? 0.f : m_used;
        const uint64_t c2 = tc::pk2(c, c), nm2 = tc::pk2(-safe, -safe);
        uint64_t l0 = 0ull, l1 = 0ull;
#pragma unroll
        for (int e = 0; e < kKeyTile / 2; e += 2) {
          const uint64_t e0 = tc::ex2_pair(tc::ffma2(tc::pk2u(x[2 * e], x[2 * e + 1]), c2, nm2), false);
          const uint64_t e1 = tc::ex2_pair(tc::ffma2(tc::pk2u(x[2 * e + 2], x[2 * e + 3]), c2, nm2), false);
          l0 = tc::fadd2(l0, e0);
          l1 = tc::fadd2(l1, e1);
          float p0, p1, p2, p3;
          tc::upk2(e0, p0, p1);
          tc::upk2(e1, p2, p3);
          x[e] = tc::pack2<T>(p0, p1);  // a slot that has been used already (e <= 2 e)
          x[e + 1] = tc::pack2<T>(p2, p3);
        }
        float a0, a1, a2, a3;
        tc::upk2(l0, a0, a1);
        tc::upk2(l1, a2, a3);
        l += (a0 + a1) + (a2 + a3);
        tc::tmem_st32(tS, x);
        if (k0 + kKeyTile > t.total) {  // rows of V behind the last key may hold anything, and 0 * NaN is NaN: they become 0
          ok = __all_sync(0xffffffffu, tc::mbar_wait(v_full + 8 * s, parity, guard, kStTilesSoftmax));
          if (!ok) break;
          const int gone = imax(t.total - k0, 0);
          for (int idx = r; idx < (kKeyTile - gone) * (DP / 8); idx += 128) {
            const int row = gone + idx / (DP / 8), u = idx % (DP / 8);
            *reinterpret_cast<uint4*>(gen + S::kV + s * S::kKvBytes + (u / 8) * S::kKvChunk + row * 128 + (u % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          tc::fence_proxy_async_smem();
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full + 8 * s);
      }
      if (ok && count > 0) ok = __all_sync(0xffffffffu, tc::mbar_wait(o_full, (uint32_t)pieces & 1u, guard, kStTilesEpilogue));
      tc::tc_fence_after();
      bool odd = i >= 0 && !(l <= 3e38f);
      const float inv = i >= 0 && l != 0.f ? 1.f / l : 0.f;
      T* to = o_row<T>(p, t.b, out_h, out_i);
      float* part = p.part_o + ((long long)piece.slot * p.rows + r) * p.D;
#pragma unroll 1
      for (int d = 0; d < DP; d += 32) {
        uint32_t o[32];
        __syncwarp();
        if (count > 0 && ok) {
          tc::tmem_ld32(tO + lane_sel + d, o);
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
          if (!piece.whole) {
            *reinterpret_cast<float4*>(part + d + e) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(part + d + e + 4) = make_float4(f[4], f[5], f[6], f[7]);
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
        if (piece.whole) store_lse(p, t.b, out_h, out_i, i >= 0, m_used, l);
        else p.part_ml[(long long)piece.slot * p.rows + r] = make_float2(m_used, l);
      }
      if (count > 0) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(o_empty);
        ++pieces;
      }
      if (consumers_any(odd)) repair_piece<T, DP, M>(p, t, piece, warp, 4);
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == 4) tc::tmem_dealloc(tmem, S::kTmemCols);
}

}  // namespace cache
}  // namespace chill
