// The tensor-core kernels multiply whole tiles: a key that a row does not see has weight 0 there, and 0 * NaN or 0 * inf is NaN.  So
// whenever a result that is not finite comes out of a piece, its rows are worked out again here, on the CUDA cores and from the
// visible keys alone.  A NaN that the visible keys do hold comes out again; finite data never gets here.
// A warp takes its rows key by key, which over a long table can take seconds (32 rows a warp by 173,000 keys: 3), longer than the
// other warps of the CTA may wait for one another.
#pragma once
#include "cache_common.cuh"
#include "tc_common.cuh"

namespace chill {
namespace cache {

// The waits of the tensor-core kernels, bounded as tc::mbar_wait's; but warps that repair are at work, not stuck, so how long a waiter waits (units of
// 2^20 ns) stands in the word behind the abort flag: kWaitLimitNs at first, and who repairs adds the time that it has taken so far.  A repair ends
// by itself after rows times keys steps, so every wait ends.
constexpr int kLimitShift = 20;
constexpr int kFirstLimit = (int)(tc::kWaitLimitNs >> kLimitShift);
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, const tc::Guard& g, int code) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((it & 7u) == 0u) {
      if (*g.abort) return false;
      const uint64_t t = tc::globaltimer_ns();
      if (t0 == 0) {
        t0 = t;
      } else if ((uint32_t)((t - t0) >> kLimitShift) > (uint32_t)g.abort[1]) {
        atomicCAS(g.status, 0, code);
        *g.abort = 1;
        return false;
      }
    }
  }
}

// Whether any of 128 threads (four warps) says so; also a barrier between their stores before and after it.
__device__ __forceinline__ bool consumers_any(bool x, int bar = 2) {
  uint32_t any;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t"
      "}\n"
      : "=r"(any)
      : "r"((uint32_t)x), "r"(bar)
      : "memory");
  return any != 0;
}

// Rows row0, row0 + warps, ... below `end` of a piece again, one row a warp, lanes over the channels, key by key.  `limit`: of the
// other warps' waits, where there are any.
template <typename T, int DP, class M, bool kMany = false>
__device__ __noinline__ void repair_piece(const CachedP& p, const RowTile& t, const Piece& piece, int row0, int warps, int end, volatile int* limit) {
  const int lane = threadIdx.x & 31;
  constexpr int kOwn = DP / 32;  // channels of a lane: lane, lane + 32, ...
  const int last = imin(t.k_lo + piece.t1 * kKeyTile, t.total);
  const uint64_t begun = tc::globaltimer_ns();
  const int before = limit != nullptr ? *limit : 0;
  for (int r = row0; r < imin(t.rows, end); r += warps) {
    const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G, pos = token_position(p, t, i);
    const T* qr = row_ptr<T>(p.q, t.b, h, i);
    float q[kOwn], o[kOwn], m = -CUDART_INF_F, l = 0.f;
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
      q[c] = lane + 32 * c < p.D ? to_f(qr[(lane + 32 * c) * p.q.sd]) : 0.f;
      o[c] = 0.f;
    }
    for (int key = t.k_lo + piece.t0 * kKeyTile; key < last; ++key) {
      if (limit != nullptr && key % kKeyTile == 0 && lane == 0) *limit = imax(*limit, before + (int)((tc::globaltimer_ns() - begun) >> kLimitShift));
      const int page = p.table[t.b * p.table_sb + key / p.page];
      if (page < 0 || page >= p.num_pages || !sees<M>(p, t, i, pos, key)) continue;
      const int row = key % p.page;
      const T* kr = reinterpret_cast<const T*>(p.k.p) + page * p.k.sb + piece.head * p.k.sh + row * p.k.sl;
      const T* vr = reinterpret_cast<const T*>(p.v.p) + page * p.v.sb + piece.head * p.v.sh + row * p.v.sl;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < kOwn; ++c)
        if (lane + 32 * c < p.D) s = fmaf(q[c], to_f(kr[(lane + 32 * c) * p.k.sd]), s);
      s = warp_sum(s) * p.scale_log2;
      const float m_new = fmaxf(m, s), safe = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float a = exp2f(m - safe), w = exp2f(s - safe);
      m = m_new;
      l = l * a + w;
#pragma unroll
      for (int c = 0; c < kOwn; ++c)
        if (lane + 32 * c < p.D) o[c] = fmaf(w, to_f(vr[(lane + 32 * c) * p.v.sd]), o[c] * a);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const long long at = (long long)piece.slot * p.rows + r;
    T* to = o_row<T>(p, t.b, h, i);
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
      const int d = lane + 32 * c;
      if (d >= p.D) continue;
      if (piece.slot < 0) to[d * p.o.sd] = from_f<T>(o[c] * inv);
      else if (kMany) p.part_o[(((long long)piece.slot * (p.D / 4) + d / 4) * p.rows + r) * 4 + d % 4] = o[c];
      else p.part_o[at * p.D + d] = o[c];
    }
    if (lane == 0) {
      if (piece.slot < 0) store_lse(p, t.b, h, i, true, m, l);
      else p.part_ml[at] = make_float2(m, l);
    }
  }
}

}  // namespace cache
}  // namespace chill
