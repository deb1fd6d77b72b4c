// Attention of FEW new tokens over a paged cache, 16-bit types: 16 or 32 rows (tokens times heads of a group) of a kv head, every key
// and value read once.  Bound by memory: 16 rows take 16 operations per byte of K and V, a B200 has about 250 to give.  So the rows
// go through mma.sync, whose tile is 16 rows (the smallest tcgen05 tile is 64, most of it would be padding, and its softmax would
// be one row a thread), and the kernel is about keeping copies in flight.
//
// A CTA (several on an SM, see rows_ctas) is one producer warp and four consumer warps:
//   producer   takes shares and hands their pieces to the consumers, two of them with their Q (a bulk copy for each row) ahead; a
//              tile is 64 keys of K and of V, boxes of `box` rows of one page and 64 channels (128-byte rows, 128B swizzle), a lane
//              for each box, into a ring of kStages tiles (48 to 192 KB a CTA).  It runs ahead into the next piece and the next share.
//   consumers  warp w takes keys 16 w .. 16 w + 15 of every tile for all rows, with a running maximum, sum and O of its own
//              in registers: no warp waits for another before the end of a piece.  S = Q K^T (B fragments of K by ldmatrix), softmax
//              on the accumulator's layout, P is the A fragment of O += P V as it stands (V by ldmatrix.trans).
//   At the end of a piece the four states are joined through shared memory, 32 channels at a time.
// For the second product the weights are 16 bits wide like V.  With 16 rows each is given as two such numbers, the rounded one and the
// rounded rest: twice the products, which the copies hide (64 requests, one token each: 180.7 us either way), and O is exact up to its own rounding.  With 32 rows once rounded, half a step of the type relative to each weight, as
// the other 16-bit kernels do (24 drafts each for 32 requests: 46.9 us, in two parts 48.5).  Sums are of the unrounded weights, in fp32.
#pragma once
#include "cache_common.cuh"
#include "cache_repair.cuh"
#include "tc_common.cuh"

namespace chill {
namespace cache {

constexpr int kRowsThreads = 256;  // warps 0-3 consumers, 4 producer, 5-7 idle

template <int DP, int MT>
struct RowsShape {
  static constexpr int kCtasPerSm = rows_ctas(DP, 16 * MT);
  // a CTA's pool is 256 threads x launch registers: consumers + others <= 2 * launch
  static constexpr int kConsumerRegs = kCtasPerSm == 3 ? 104 : 184, kOtherRegs = kCtasPerSm == 3 ? 56 : 72;
  static_assert(kCtasPerSm == 1 || kConsumerRegs + kOtherRegs <= 2 * (65536 / (256 * kCtasPerSm) / 8 * 8), "setmaxnreg.inc would never be granted");
  static constexpr int kHalves = DP / 64;                      // 64-channel blocks
  static constexpr int kTileBytes = kKeyTile * DP * 2;         // K or V
  static constexpr int kStages = DP == 64 ? (kCtasPerSm == 3 ? 3 : 5) : (MT == 1 ? 3 : 2);  // what the CTAs of an SM have room for
  static constexpr int kRows = 16 * MT;
  static constexpr int kQPitch = DP * 2 + 16;                  // bytes of a row of Q: eight rows in different banks
  static constexpr int kQBytes = kRows * kQPitch;
  static constexpr int kMergeBytes = 4 * 16 * 32 * 4;          // four warps, 16 rows, 32 channels
  static constexpr int kRing = 0;                              // stage: K, then V
  // Two Q, what the merge buffer is longer than a Q between them: it lies over the Q that has been used, and over that
  static constexpr int kQ = kStages * 2 * kTileBytes;
  static constexpr int kBetween = kMergeBytes > kQBytes ? kMergeBytes - kQBytes : 0;
  static constexpr int kStat = kQ + 2 * kQBytes + kBetween;    // maximum and sum of each warp's rows
  static constexpr int kBars = kStat + 4 * kRows * 8;          // full[stage], empty[stage], item_full[2], item_empty[2]
  static constexpr int kHoles = kBars + (2 * kStages + 4) * 8; // groups of 8 keys without a page, a word per stage
  static constexpr int kMisc = kHoles + kStages * 4;            // abort flag, limit of the waits
  static constexpr int kItems = (kMisc + 16 + 15) / 16 * 16;
  static constexpr int kCum = kItems + 2 * (int)sizeof(Item);
  static constexpr int kTotal = kCum + (kScanEntries + 1) * 4;
  static constexpr int kDynamic = kTotal + 1024;               // slack for manual 1024-byte alignment
  static_assert(kCtasPerSm * (kDynamic + 1024) <= 233472, "shared memory of an SM");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// size bytes (a multiple of 16) from global to shared memory, both on 16-byte boundaries.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t size, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(size), "r"(bar) : "memory");
}

enum : int { kStRowsProducer = 701, kStRowsConsumer = 702 };

template <typename T, int DP, int MT, class M>
__global__ void __launch_bounds__(kRowsThreads, RowsShape<DP, MT>::kCtasPerSm)
cached_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CachedP p) {
  using S = RowsShape<DP, MT>;
  constexpr int kStages = S::kStages;
  constexpr bool kTwoParts = MT == 1;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - tc::smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full = base + S::kBars, empty = full + 8 * kStages, item_full = empty + 8 * kStages, item_empty = item_full + 16;
  volatile int* holes = reinterpret_cast<volatile int*>(gen + S::kHoles);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + S::kMisc);
  Item* items = reinterpret_cast<Item*>(gen + S::kItems);
  const tc::Guard guard{p.status, abort_flag};
  if (threadIdx.x == 0) {
    abort_flag[0] = 0;
    abort_flag[1] = kFirstLimit;
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(full + 8 * s, 1);
      tc::mbar_init(empty + 8 * s, 4);
    }
    for (int s = 0; s < 2; ++s) {
      tc::mbar_init(item_full + 8 * s, 1);
      tc::mbar_init(item_empty + 8 * s, 4);
    }
    tc::fence_barrier_init();
  }
  // channels of Q beyond the head stay 0: those of K are filled with zeros, and 0 * NaN is NaN
  if (p.D < DP)
    for (int idx = threadIdx.x; idx < (2 * S::kQBytes + S::kBetween) / 16; idx += kRowsThreads) *reinterpret_cast<uint4*>(gen + S::kQ + idx * 16) = make_uint4(0u, 0u, 0u, 0u);
  tc::fence_proxy_async_smem();
  const int* cum;
  const Cut cut = begin_work<M, kRowsThreads>(p, reinterpret_cast<int*>(gen + S::kCum), cum);
  __syncthreads();
  pdl_launch_dependents();

  if (warp >= 4) {
    if constexpr (S::kCtasPerSm > 1) tc::reg_dealloc<S::kOtherRegs>();
    if (warp > 4) return;
    // ---------------------------------------------------------------------------------------------- producer
    const int boxes = kKeyTile / p.box, jobs = boxes * S::kHalves, mine = lane % boxes;
    const uint32_t box_bytes = (uint32_t)p.box * 128u;
    int n = 0;  // tiles so far
    bool ok = true;
    Work work;
    work.start<M>(p, cut, cum);
    Item it;
    for (int item = 0;; ++item) {
      const bool more = work.next<M>(p, it);
      const int slot = item & 1;
      ok = __all_sync(0xffffffffu, bounded_wait(item_empty + 8 * slot, ((uint32_t)(item >> 1) & 1u) ^ 1u, guard, kStRowsProducer));
      if (!ok) break;
      const RowTile& t = it.t;
      const uint32_t sq = base + S::kQ + slot * (S::kQBytes + S::kBetween), bar = item_full + 8 * slot;
      if (more && it.tiles > 0 && !p.wide_q) {  // rows of Q that can not be copied in bulk
        for (int idx = lane; idx < t.rows * p.D; idx += 32) {
          const int r = idx / p.D, d = idx - r * p.D, i = (t.r0 + r) / p.G, h = it.x.head * p.G + (t.r0 + r) % p.G;
          *reinterpret_cast<T*>(gen + (sq - base) + r * S::kQPitch + d * 2) = row_ptr<T>(p.q, t.b, h, i)[d * p.q.sd];
        }
        __syncwarp();
      }
      const bool bulk = more && it.tiles > 0 && p.wide_q;
      if (lane == 0) {
        items[slot] = it;
        if (bulk) tc::mbar_arrive_expect_tx(bar, (uint32_t)(t.rows * p.D * 2));
        else tc::mbar_arrive(bar);
      }
      __syncwarp();
      if (!more) break;
      if (bulk && lane < t.rows) {
        const int i = (t.r0 + lane) / p.G, h = it.x.head * p.G + (t.r0 + lane) % p.G;
        bulk_load(sq + lane * S::kQPitch, row_ptr<T>(p.q, t.b, h, i), (uint32_t)(p.D * 2), bar);
      }
      bool there = false, there_next = false;
      int page = 0, page_next = 0;
      if (it.x.t0 < it.tiles) page_next = tile_page(p, t, t.k_lo + it.x.t0 * kKeyTile, mine, there_next);
      for (int kt = it.x.t0; kt < it.tiles; ++kt, ++n) {
        const int s = n % kStages, k0 = t.k_lo + kt * kKeyTile;
        page = page_next;
        there = there_next;
        if (kt + 1 < it.tiles) page_next = tile_page(p, t, k0 + kKeyTile, mine, there_next);
        const unsigned lost = __ballot_sync(0xffffffffu, !there && lane < boxes);
        ok = __all_sync(0xffffffffu, bounded_wait(empty + 8 * s, ((uint32_t)(n / kStages) & 1u) ^ 1u, guard, kStRowsProducer));
        if (!ok) break;
        if (lane == 0) {
          holes[s] = lost_groups(p, lost, boxes);
          tc::mbar_arrive_expect_tx(full + 8 * s, 2 * S::kTileBytes);
        }
        __syncwarp();
        const int row = (k0 + mine * p.box) % p.page;
        for (int j = lane; j < jobs; j += 32) {
          const int half = j / boxes;
          const uint32_t dst = base + S::kRing + s * 2 * S::kTileBytes + half * (kKeyTile * 128) + mine * box_bytes;
          tc::tma_load_4d(dst, &tmK, full + 8 * s, half * 64, row, it.x.head, page);
          tc::tma_load_4d(dst + S::kTileBytes, &tmV, full + 8 * s, half * 64, row, it.x.head, page);
        }
      }
      if (!ok) break;
    }
    if (!ok) {  // copies already in flight land before the CTA's shared memory goes away
      const uint64_t t0 = tc::globaltimer_ns();
      while (tc::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    return;
  }

  // ------------------------------------------------------------------------------------------------- consumers
  if constexpr (S::kCtasPerSm > 1) tc::reg_alloc<S::kConsumerRegs>();
  const int g = lane >> 2, quad = lane & 3;  // the accumulator's rows g and g + 8, channels / keys 2 quad, 2 quad + 1 of 8
  float2* stat = reinterpret_cast<float2*>(gen + S::kStat);
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int item = 0;; ++item) {
    const int slot = item & 1;
    // The four warps leave together: whether there is one more piece, and whether all of them saw it, is settled at a barrier
    bool leave = !__all_sync(0xffffffffu, bounded_wait(item_full + 8 * slot, (uint32_t)(item >> 1) & 1u, guard, kStRowsConsumer));
    if (!leave) leave = items[slot].x.entry < 0;
    if (consumers_any(leave)) break;
    const RowTile& t = items[slot].t;
    const Piece& piece = items[slot].x;
    const int tiles = items[slot].tiles, k_lo = t.k_lo, total = t.total, full_lo = t.full_lo, full_hi = t.full_hi;
    const uint32_t sq = base + S::kQ + slot * (S::kQBytes + S::kBetween);
    float* merge = reinterpret_cast<float*>(gen + S::kQ + slot * S::kQBytes);
    const int row_token = lane < t.rows ? (t.r0 + lane) / p.G : -1;  // of row `lane`
    const int row_pos = lane < t.rows ? token_position(p, t, row_token) : 0;
    const uint64_t row_near = first_ancestors(p, t.b, row_token);

    float o[MT][DP / 8][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt][0] = m[mt][1] = -CUDART_INF_F;
      l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) o[mt][c][0] = o[mt][c][1] = o[mt][c][2] = o[mt][c][3] = 0.f;
    }
    // this lane's row of the fragments: ldmatrix takes the address of row lane % 8 of matrix lane / 8
    const int q_row = ((lane >> 3) & 1) * 8 + (lane & 7), q_unit = lane >> 4;
    const int k_row = warp * 16 + (lane >> 4) * 8 + (lane & 7), k_unit = (lane >> 3) & 1;
    const int v_row = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), v_unit = lane >> 4;
    const int x7 = lane & 7;  // row % 8 in all three

    for (int kt = piece.t0; kt < tiles; ++kt) {
      const int s = stage, k0 = k_lo + kt * kKeyTile;
      const uint32_t sk = base + S::kRing + s * 2 * S::kTileBytes, sv = sk + S::kTileBytes;
      ok = __all_sync(0xffffffffu, bounded_wait(full + 8 * s, phase, guard, kStRowsConsumer));
      if (!ok) break;  // the rest of the piece is skipped; the next one's wait fails at once
      float c[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 2; ++j) c[mt][j][0] = c[mt][j][1] = c[mt][j][2] = c[mt][j][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t b[4];
        ldsm4(b, sk + (kk / 4) * (kKeyTile * 128) + k_row * 128 + ((((kk % 4) * 2 + k_unit) ^ x7) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a[4];
          ldsm4(a, sq + (mt * 16 + q_row) * S::kQPitch + (kk * 2 + q_unit) * 16);
          mma16816<T>(c[mt][0], a, b[0], b[1]);
          mma16816<T>(c[mt][1], a, b[2], b[3]);
        }
      }
      const int lost = holes[s];
      if (lost != 0 || k0 < full_lo || k0 + kKeyTile > full_hi) {
        // lane r works out row r's keys; a thread then takes those of its own rows
        uint64_t vis = visible_keys<M>(p, t, row_token, row_pos, row_near, k0, lost);
        __syncwarp();
        const uint32_t half = warp < 2 ? (uint32_t)vis : (uint32_t)(vis >> 32);  // the 32 keys that hold this warp's 16
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t mine = __shfl_sync(0xffffffffu, half, mt * 16 + g + 8 * u) >> ((warp & 1) * 16 + quad * 2);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (((mine >> (j * 8 + e)) & 1u) == 0u) c[mt][j][u * 2 + e] = -CUDART_INF_F;
          }
        if (k0 + kKeyTile > total) {  // rows behind the last key may hold anything, and 0 * NaN is NaN: this warp's become 0
          const int gone = imax(total - k0, 0);
          for (int idx = lane; idx < 16 * (DP / 8); idx += 32) {
            const int r = warp * 16 + idx / (DP / 8), unit = idx % (DP / 8);
            if (r >= gone) *reinterpret_cast<uint4*>(gen + (sv - base) + (unit / 8) * (kKeyTile * 128) + r * 128 + (unit % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          tc::fence_proxy_async_smem();  // the next copy into this stage comes behind these writes
          __syncwarp();
        }
      }
      // All rows' maxima first, then one look whether any of them moved far: the rows' chains run side by side
      float top[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) top[mt][u] = fmaxf(fmaxf(c[mt][0][2 * u], c[mt][0][2 * u + 1]), fmaxf(c[mt][1][2 * u], c[mt][1][2 * u + 1]));
#pragma unroll
      for (int x = 1; x <= 2; x <<= 1)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) top[mt][u] = fmaxf(top[mt][u], __shfl_xor_sync(0xffffffffu, top[mt][u], x));
      bool far = false;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          top[mt][u] *= p.scale_log2;
          far |= top[mt][u] - m[mt][u] > 8.f;
        }
      // The maximum is followed lazily: O is rescaled when it grew by more than 2^8 (weights stay below that, exact in fp32 sums and far
      // from the 16-bit types' limits), so most tiles do not touch O
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // a row goes by itself: rows that do not exist hold anything
            const bool moves = top[mt][u] - m[mt][u] > 8.f;
            const float a = moves ? tc::ex2(m[mt][u] - top[mt][u]) : 1.f;
            m[mt][u] = moves ? top[mt][u] : m[mt][u];
            l[mt][u] *= a;
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) o[mt][d][2 * u] *= a, o[mt][d][2 * u + 1] *= a;
          }
      }
      uint32_t pa[MT][4], rest[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float safe = m[mt][u] == -CUDART_INF_F ? 0.f : m[mt][u];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float w0 = tc::ex2(fmaf(c[mt][j][2 * u], p.scale_log2, -safe)), w1 = tc::ex2(fmaf(c[mt][j][2 * u + 1], p.scale_log2, -safe));
            l[mt][u] += w0 + w1;
            pa[mt][j * 2 + u] = tc::pack2<T>(w0, w1);
            if (kTwoParts) {
              float h0, h1;
              tc::unpack2<T>(pa[mt][j * 2 + u], h0, h1);
              rest[mt][j * 2 + u] = tc::pack2<T>(w0 - h0, w1 - h1);
            }
          }
        }
#pragma unroll
      for (int nn = 0; nn < DP / 16; ++nn) {
        uint32_t b[4];
        ldsm4_t(b, sv + (nn / 4) * (kKeyTile * 128) + v_row * 128 + ((((nn % 4) * 2 + v_unit) ^ x7) << 4));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<T>(o[mt][2 * nn], pa[mt], b[0], b[1]);
          mma16816<T>(o[mt][2 * nn + 1], pa[mt], b[2], b[3]);
          if (kTwoParts) {
            mma16816<T>(o[mt][2 * nn], rest[mt], b[0], b[1]);
            mma16816<T>(o[mt][2 * nn + 1], rest[mt], b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(empty + 8 * s);
      if (++stage == kStages) stage = 0, phase ^= 1u;
    }

    // ---- the four warps' states become one
    bool odd = false;  // a result that is not finite: hidden keys may have let theirs in
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 1);
        l[mt][u] += __shfl_xor_sync(0xffffffffu, l[mt][u], 2);
        if (quad == 0) stat[warp * S::kRows + mt * 16 + g + 8 * u] = make_float2(m[mt][u], l[mt][u]);
      }
    tc::named_bar_sync(1, 128);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = mt * 16 + g + 8 * u;
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w * S::kRows + r].x);
        const float a = top == -CUDART_INF_F ? 0.f : tc::ex2(m[mt][u] - top);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) o[mt][d][2 * u] *= a, o[mt][d][2 * u + 1] *= a;
      }
    const int out_r = threadIdx.x >> 3, out_c = (threadIdx.x & 7) * 4;  // this thread's row and channels of a 16 x 32 block
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = mt * 16 + out_r, all_rows = p.N * p.G;
      float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w * S::kRows + r].x);
      if (top != -CUDART_INF_F) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 x = stat[w * S::kRows + r];
          sum += tc::ex2(x.x - top) * x.y;
        }
      }
      const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
      const float inv = r < t.rows && sum != 0.f ? 1.f / sum : 0.f;
      odd |= r < t.rows && !(fabsf(sum) <= 3e38f);
#pragma unroll
      for (int cb = 0; cb < DP / 32; ++cb) {
        tc::named_bar_sync(1, 128);
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            *reinterpret_cast<float2*>(merge + (warp * 16 + g + 8 * u) * 32 + ((d ^ (g & 3)) * 8) + quad * 2) = make_float2(o[mt][cb * 4 + d][2 * u], o[mt][cb * 4 + d][2 * u + 1]);
        tc::named_bar_sync(1, 128);
        const int swizzled = out_c ^ ((out_r & 3) * 8);  // rows that lie 128 bytes apart are stored from different banks
        float4 x = *reinterpret_cast<const float4*>(merge + out_r * 32 + swizzled);
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          const float4 y = *reinterpret_cast<const float4*>(merge + (w * 16 + out_r) * 32 + swizzled);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        const int ch = cb * 32 + out_c;
        if (ch >= p.D || t.r0 + r >= all_rows) continue;
        odd |= r < t.rows && !(fabsf(x.x) + fabsf(x.y) + fabsf(x.z) + fabsf(x.w) <= 3e38f);
        if (piece.slot < 0) {
          T* to = o_row<T>(p, t.b, h, i);
          if (r >= t.rows) x = make_float4(0.f, 0.f, 0.f, 0.f);
          store4<T>(p, to, ch, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        } else {
          *reinterpret_cast<float4*>(p.part_o + ((long long)piece.slot * p.rows + r) * p.D + ch) = x;
        }
      }
      if (out_c == 0 && t.r0 + r < all_rows) {
        if (piece.slot < 0) store_lse(p, t.b, h, i, r < t.rows, top, sum);
        else p.part_ml[(long long)piece.slot * p.rows + r] = make_float2(top, sum);
      }
    }
    if (consumers_any(odd)) repair_piece<T, DP, M>(p, t, piece, warp, 4, S::kRows, abort_flag + 1);
    if (p.D < DP) {  // the channels beyond the head become 0 again
      tc::named_bar_sync(1, 128);
      for (int idx = threadIdx.x; idx < S::kQBytes / 16; idx += 128) *reinterpret_cast<uint4*>(gen + (sq - base) + idx * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    tc::fence_proxy_async_smem();  // the merge buffer and these zeros lie where the next copy of Q goes
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(item_empty + 8 * slot);
  }
}

}  // namespace cache
}  // namespace chill
