// Attention of new tokens over a paged cache on the CUDA cores: fp32 (IEEE arithmetic) and every layout that the tensor-core
// kernels can not take.  See cache_common.cuh for units and shares.
//
// Few rows (simt_few, tiles of 2 or 4): bound by memory, so nothing goes through shared memory but the weights.  D / 4 lanes (32 at most)
// share a key, a warp has 16 keys of every tile of 64; a lane keeps four channels (eight at head dim 256) of Q and O of every row and
// reads those of K and V of eight steps at once.  The 16 or 32 scores of such a batch are summed over the lanes all together: lanes halve what they
// hold at each step, each ends up with one or two scores, keeps the maximum and the sum of that row, and takes the exponential once.  Every group
// of lanes has a state of its own: no warp, and no group, waits for another before the end of a piece.
// fp32, one new token for 64 requests of up to 4000, 16 heads on 4 of 128: 127 us; with every score summed in all lanes and two CTAs on an SM
// 206; with that sum and two CTAs 192, three 177, four (128 registers) 127, six with batches of half the size 133.
// 8 heads on 8 of 128: 222 us (4.9 TB/s); in tiles of 4 rows and with sums in all lanes 416.
// More rows (simt_many): bound by the FMAs and what they read from shared memory, so a thread has a block of both products.  A CTA of 128
// threads, 16 across and 8 down, works on 8 RT rows (8, 16 or 32) and 64 keys at a time, everything as fp32 in shared memory:
//   S = Q K^T   a thread has RT rows and 4 keys: RT + 4 vectors read for 16 RT FMAs, two at a time (even and odd channels)
//   softmax     the 16 threads of a row agree on its maximum by butterflies; each keeps a sum of its own to the end
//   O += P V    a thread has RT rows and D / 16 channels; P goes through shared memory, between threads of one warp only
// K of the next tile is copied during the second product, V of this one during the first (asynchronous copies where the rows are fp32 on
// 16-byte boundaries).  Vectors are put at chunk ^ (key mod 8) of a row, so that the reads of a warp fall into different banks.
// fp32, 500 new tokens for 2 requests of up to 4000, 16 heads on 4 of 128: 1113 us, 25 TFLOP/s (an SM reads as long as it multiplies); 12 drafts
// for 8 requests of up to 5000 tokens, 16 heads on 8 of 128: 137 us.  (One key and 8 rows a thread, nothing copied ahead: 3016 and 427 us.)
// (make_plan has which rows go where.)
#pragma once
#include "cache_common.cuh"
#include "cache_repair.cuh"
#include "tc_common.cuh"

namespace chill {
namespace cache {

constexpr int kSimtThreads = 128;

template <int DP, int RT>
struct SimtSmem {  // in floats
  static constexpr int kRows = 8 * RT;
  static constexpr int kCtasPerSm = DP <= 64 ? 4 : (DP <= 128 ? 2 : 1);
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kRows * DP;
  static constexpr int kV = kK + kKeyTile * DP;
  static constexpr int kP = kV + kKeyTile * DP;
  static constexpr int kPlaces = kP + kRows * kKeyTile;  // page and row of every key of a tile, of two tiles
  static constexpr int kThere = kPlaces + 4 * kKeyTile;  // a bit for every key: it has a page
  static constexpr int kItem = kThere + 4;
  static constexpr int kCum = kItem + (int)sizeof(Item) / 4;
  static constexpr int kBytes = (kCum + kScanEntries + 1) * 4;
};

__device__ __forceinline__ void copy16(float* dst, const void* src, bool there) {  // zeros where there is nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Four channels from global memory, as fp32.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, long long sd, bool wide) {
  if (wide) {
    if constexpr (sizeof(T) == 4) {
      return *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      float4 f;
      tc::unpack2<T>(x.x, f.x, f.y);
      tc::unpack2<T>(x.y, f.z, f.w);
      return f;
    }
  }
  return make_float4(to_f(p[0]), to_f(p[sd]), to_f(p[2 * sd]), to_f(p[3 * sd]));
}

template <typename T, int DP, int RT, class M>
__global__ void __launch_bounds__(kSimtThreads, (SimtSmem<DP, RT>::kCtasPerSm)) cached_simt_many_kernel(const __grid_constant__ CachedP p) {
  using L = SimtSmem<DP, RT>;
  constexpr int kChunks = DP / 4, kVecs = DP > 64 ? DP / 64 : 1;
  extern __shared__ __align__(16) float smem[];
  float *sq = smem + L::kQ, *sk = smem + L::kK, *sv = smem + L::kV, *sp = smem + L::kP;
  int2* places = reinterpret_cast<int2*>(smem + L::kPlaces);
  volatile unsigned* there = reinterpret_cast<volatile unsigned*>(smem + L::kThere);
  Item& item = *reinterpret_cast<Item*>(smem + L::kItem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tx = tid & 15, ty = tid >> 4, odd_row = ty & 1;
  const int* cum;
  const Cut cut = begin_work<M, kSimtThreads>(p, reinterpret_cast<int*>(smem + L::kCum), cum);
  pdl_launch_dependents();
  Work work;
  if (warp == 0) work.start<M>(p, cut, cum);
  while (true) {
    __syncthreads();
    if (warp == 0) {
      Item it;
      work.next<M>(p, it);
      if (lane == 0) item = it;
    }
    __syncthreads();
    if (item.x.entry < 0) break;
    const RowTile& t = item.t;
    const Piece& piece = item.x;
    const int tiles = item.tiles, t0 = piece.t0, total = t.total, k_lo = t.k_lo, full_lo = t.full_lo, full_hi = t.full_hi;
    // page and row of this thread's key of a tile
    auto place = [&](int kt) -> int2 {
      const int at = k_lo + kt * kKeyTile + tid, block = at / p.page;
      const int page = at < total ? p.table[t.b * p.table_sb + block] : -1;
      return make_int2(page >= 0 && page < p.num_pages ? page : -1, at - block * p.page);
    };
    auto put_place = [&](int kt, int2 x) {
      places[((kt - t0) & 1) * kKeyTile + tid] = x;
      const unsigned is = __ballot_sync(0xffffffffu, x.x >= 0);
      if (lane == 0) there[((kt - t0) & 1) * 2 + warp] = is;
    };
    auto copy = [&](int kt, const TRef& c, float* to, bool swizzle) {  // K or V of a tile
#pragma unroll 4
      for (int idx = tid; idx < kKeyTile * kChunks; idx += kSimtThreads) {
        const int key = idx / kChunks, ch = idx % kChunks;
        const int2 x = places[((kt - t0) & 1) * kKeyTile + key];
        const bool is = x.x >= 0 && ch * 4 < p.D;
        const T* from = reinterpret_cast<const T*>(c.p) + (is ? x.x * c.sb + piece.head * c.sh + x.y * c.sl + ch * 4 * c.sd : 0);
        float* dst = to + key * DP + (swizzle ? ch ^ (key & 7) : ch) * 4;
        if (sizeof(T) == 4 && p.wide_kv) copy16(dst, from, is);
        else *reinterpret_cast<float4*>(dst) = is ? load4<T>(from, c.sd, p.wide_kv) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    if (t0 < tiles && tid < kKeyTile) put_place(t0, place(t0));
    for (int idx = tid; idx < L::kRows * kChunks; idx += kSimtThreads) {
      const int r = idx / kChunks, ch = idx % kChunks;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < t.rows && ch * 4 < p.D) {
        const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
        x = load4<T>(row_ptr<T>(p.q, t.b, h, i) + ch * 4 * p.q.sd, p.q.sd, p.wide_q);
      }
      *reinterpret_cast<float4*>(sq + r * DP + (ch ^ (r / RT & 1)) * 4) = x;
    }
    // of row ty * RT + tx, where there is one
    const int my_row = tx < RT ? ty * RT + tx : -1, my_token = my_row >= 0 && my_row < t.rows ? (t.r0 + my_row) / p.G : -1;
    const int my_pos = my_token >= 0 ? token_position(p, t, my_token) : 0;
    const uint64_t my_near = first_ancestors(p, t.b, my_token);
    float m[RT], l[RT];  // the maximum is the same in the 16 threads of a row, the sum each one's own
    uint64_t o[RT][kVecs][2];
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      m[n] = -CUDART_INF_F;
      l[n] = 0.f;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) o[n][v][0] = o[n][v][1] = 0ull;
    }
    __syncthreads();
    if (t0 < tiles) copy(t0, p.k, sk, true);
    for (int kt = t0; kt < tiles; ++kt) {
      const int k0 = k_lo + kt * kKeyTile;
      const bool more = kt + 1 < tiles;
      int2 next = make_int2(-1, 0);
      if (more && tid < kKeyTile) next = place(kt + 1);
      copies_done();
      __syncthreads();  // K is there; V of the tile before has been used
      copy(kt, p.v, sv, false);
      uint64_t s2[RT][4];
#pragma unroll
      for (int n = 0; n < RT; ++n) s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0ull;
#pragma unroll 4
      for (int ch = 0; ch < kChunks; ++ch) {
        ulonglong2 q[RT], k[4];
#pragma unroll
        for (int n = 0; n < RT; ++n) q[n] = *reinterpret_cast<const ulonglong2*>(sq + (ty * RT + n) * DP + (ch ^ odd_row) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const ulonglong2*>(sk + (tx + 16 * j) * DP + (ch ^ (tx & 7)) * 4);
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s2[n][j] = tc::ffma2(q[n].y, k[j].y, tc::ffma2(q[n].x, k[j].x, s2[n][j]));
      }
      const unsigned th0 = there[((kt - t0) & 1) * 2], th1 = there[((kt - t0) & 1) * 2 + 1];
      const bool full = (th0 & th1) == 0xffffffffu && k0 >= full_lo && k0 + kKeyTile <= full_hi;
      uint64_t vis = ~0ull;
      if (!full) {
        vis = visible_keys<M>(p, t, my_token, my_pos, my_near, k0, 0) & ((uint64_t)th0 | (uint64_t)th1 << 32);
        __syncwarp();
      }
#pragma unroll
      for (int n = 0; n < RT; ++n) {
        const uint64_t see = full ? ~0ull : __shfl_sync(0xffffffffu, (unsigned long long)vis, (lane & 16) + n);
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float lo, hi;
          tc::upk2(s2[n][j], lo, hi);
          x[j] = (see >> (tx + 16 * j)) & 1ull ? (lo + hi) * p.scale_log2 : -CUDART_INF_F;
        }
        float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float m_new = fmaxf(m[n], top), safe = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float a = exp2f(m[n] - safe);  // m = -inf: 0
        m[n] = m_new;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = exp2f(x[j] - safe);
          sp[(ty * RT + n) * kKeyTile + ((tx + 16 * j) ^ (odd_row * 16))] = x[j];
        }
        l[n] = fmaf(l[n], a, (x[0] + x[1]) + (x[2] + x[3]));
        if (a != 1.f) {
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            o[n][v][0] = tc::fmul2(o[n][v][0], tc::pk2(a, a));
            o[n][v][1] = tc::fmul2(o[n][v][1], tc::pk2(a, a));
          }
        }
      }
      if (more && tid < kKeyTile) put_place(kt + 1, next);
      copies_done();
      __syncthreads();  // V is there; K has been used
      if (more) copy(kt + 1, p.k, sk, true);
      if (DP >= 64 || tx * 4 < DP) {
#pragma unroll 2
        for (int k4 = 0; k4 < kKeyTile; k4 += 4) {
          float4 w[RT];
#pragma unroll
          for (int n = 0; n < RT; ++n) w[n] = *reinterpret_cast<const float4*>(sp + (ty * RT + n) * kKeyTile + (k4 ^ (odd_row * 16)));
#pragma unroll
          for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
              const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(sv + (k4 + u) * DP + v * 64 + tx * 4);
#pragma unroll
              for (int n = 0; n < RT; ++n) {
                const float wn = u == 0 ? w[n].x : (u == 1 ? w[n].y : (u == 2 ? w[n].z : w[n].w));
                o[n][v][0] = tc::ffma2(tc::pk2(wn, wn), x.x, o[n][v][0]);
                o[n][v][1] = tc::ffma2(tc::pk2(wn, wn), x.y, o[n][v][1]);
              }
            }
          }
        }
      }
    }

    bool odd = false;  // not finite: a hidden key's 0 times what it holds, maybe
#pragma unroll
    for (int n = 0; n < RT; ++n) {
      const int r = ty * RT + n;
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], d);
      if (t.r0 + r >= p.N * p.G) continue;
      const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
      const long long at = (long long)imax(piece.slot, 0) * p.rows + r;
      const bool valid = r < t.rows;
      const float inv = l[n] != 0.f ? 1.f / l[n] : 0.f;
      T* to = o_row<T>(p, t.b, h, i);
      odd |= valid && !(l[n] <= 3e38f);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int d = v * 64 + tx * 4;
        if (d >= p.D || (DP < 64 && d >= DP)) continue;
        float f[4];
        tc::upk2(o[n][v][0], f[0], f[1]);
        tc::upk2(o[n][v][1], f[2], f[3]);
        odd |= valid && !(fabsf(f[0]) + fabsf(f[1]) + fabsf(f[2]) + fabsf(f[3]) <= 3e38f);
        if (piece.slot >= 0) *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = make_float4(f[0], f[1], f[2], f[3]);
        else if (valid) store4<T>(p, to, d, f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
        else store4<T>(p, to, d, 0.f, 0.f, 0.f, 0.f);
      }
      if (tx == 0) {
        if (piece.slot >= 0) p.part_ml[at] = make_float2(m[n], l[n]);
        else store_lse(p, t.b, h, i, valid, m[n], l[n]);
      }
    }
    if (consumers_any(odd)) repair_piece<T, DP, M>(p, t, piece, warp, 4, L::kRows, nullptr);
  }
}

// Sums N values over 2 STEP lanes, which halve the values that they hold at each step: lane `sub` of them ends up with those from
// sub * N / (2 STEP) on, or, where there are fewer values than lanes, with the one it shares with its neighbours.
template <int N, int STEP>
__device__ __forceinline__ void lane_sums(float* x, int sub) {
  if constexpr (N > 1) {
    const bool upper = (sub & STEP) != 0;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float keep = upper ? x[i + N / 2] : x[i], give = upper ? x[i] : x[i + N / 2];
      x[i] = keep + __shfl_xor_sync(0xffffffffu, give, STEP);
    }
  } else {
    x[0] += __shfl_xor_sync(0xffffffffu, x[0], STEP);
  }
  if constexpr (STEP > 1) lane_sums<(N > 1 ? N / 2 : 1), STEP / 2>(x, sub);
}

// WARPS: four of them have a tile; with eight (units taken whole, where one CTA has all of a unit's tiles) two tiles are under way.
template <typename T, int DP, int R, int WARPS, class M>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) cached_simt_few_kernel(const __grid_constant__ CachedP p) {
  constexpr int kLanes = DP / 4 < 32 ? DP / 4 : 32;     // of a key
  constexpr int kVecs = DP / 4 / kLanes;                // vectors of four channels of a lane
  constexpr int kKeys = 32 / kLanes;                    // keys of a warp at a time: its groups of lanes
  constexpr int kSteps = 16 / kKeys;                    // of the warp's 16 keys of a tile
  constexpr int kAhead = kSteps < 8 / kVecs ? kSteps : 8 / kVecs;  // steps whose loads are in flight
  constexpr int kVals = R * kAhead, kOwn = kVals > kLanes ? kVals / kLanes : 1;  // scores of such a batch, and how many a lane ends up with
  constexpr int kSame = kVals < kLanes ? kLanes / kVals : 1, kRowLanes = kLanes / R;  // lanes with the same score; lanes of a row
  __shared__ float4 sums[WARPS][R][DP / 4];
  __shared__ float4 weights[WARPS][kKeys][kVals / 4];
  __shared__ float alpha[WARPS][kKeys][R];
  __shared__ float2 stat[WARPS][R];
  __shared__ Item item;
  __shared__ int smem_cum[kScanEntries + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = lane / kLanes, ch = (lane % kLanes) * 4;
  const int* cum;
  const Cut cut = begin_work<M, WARPS * 32>(p, smem_cum, cum);
  pdl_launch_dependents();
  Work work;
  if (warp == 0) work.start<M>(p, cut, cum);
  while (true) {
    __syncthreads();
    if (warp == 0) {
      Item it;
      work.next<M>(p, it);
      if (lane == 0) item = it;
    }
    __syncthreads();
    if (item.x.entry < 0) break;
    const RowTile& t = item.t;
    const Piece piece = item.x;
    const int tiles = item.tiles, total = t.total, rows = t.rows, k_lo = t.k_lo, full_lo = t.full_lo, full_hi = t.full_hi;
    float4 q[R][kVecs], o[R][kVecs];
    const int sub = lane % kLanes, my_r = sub / kRowLanes;  // this lane's row, and its maximum and part of the sum
    float my_m = -CUDART_INF_F, my_l = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const int d = ch + v * 128;
        q[r][v] = o[r][v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && d < p.D) {
          const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
          q[r][v] = load4<T>(row_ptr<T>(p.q, t.b, h, i) + d * p.q.sd, p.q.sd, p.wide_q);
        }
      }
    }
    const int* table = p.table + t.b * p.table_sb;
    const int my_token = lane < rows ? (t.r0 + lane) / p.G : -1, my_pos = lane < rows ? token_position(p, t, my_token) : 0;  // of row `lane`
    const uint64_t my_near = first_ancestors(p, t.b, my_token);
    const char* kb = reinterpret_cast<const char*>(p.k.p) + (piece.head * p.k.sh + ch * p.k.sd) * (long long)sizeof(T);
    const char* vb = reinterpret_cast<const char*>(p.v.p) + (piece.head * p.v.sh + ch * p.v.sd) * (long long)sizeof(T);
    const int quarter = (warp & 3) * 16;  // this warp's keys of a tile
    auto page_of = [&](int k) -> int {  // of key k + lane, for the first 16 lanes
      const int page = lane < 16 && k + lane < total ? table[(k + lane) / p.page] : -1;
      return page < p.num_pages ? page : -1;
    };
    int pages_next = page_of(k_lo + (piece.t0 + warp / 4) * kKeyTile + quarter);
    for (int kt = piece.t0 + warp / 4; kt < tiles; kt += WARPS / 4) {
      const int k0 = k_lo + kt * kKeyTile + quarter, pages = pages_next;
      pages_next = page_of(k0 + WARPS / 4 * kKeyTile);
      if (k0 >= total) break;
      unsigned seen = my_r < rows ? 0xffffu : 0u;  // bit s * kKeys + g: row my_r sees the key of group g in step s
      if (k0 < full_lo || k0 + 16 > full_hi) {
        const uint64_t vis = visible_keys<M>(p, t, my_token, my_pos, my_near, k0 - quarter, 0);
        __syncwarp();
        seen = __shfl_sync(0xffffffffu, (unsigned)(vis >> quarter), my_r);  // what lane r holds is row r's
      }
#pragma unroll 1
      for (int s0 = 0; s0 < kSteps; s0 += kAhead) {
        float4 kx[kAhead][kVecs], vx[kAhead][kVecs];
        unsigned there = 0;
        int row = (k0 + s0 * kKeys + group) % p.page;
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
          const int page = __shfl_sync(0xffffffffu, pages, (s0 + s) * kKeys + group);
          const bool is = page >= 0;
          there |= (unsigned)is << s;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            kx[s][v] = vx[s][v] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (is && ch + v * 128 < p.D) {
              kx[s][v] = load4<T>(reinterpret_cast<const T*>(kb) + page * p.k.sb + row * p.k.sl + v * 128 * p.k.sd, p.k.sd, p.wide_kv);
              vx[s][v] = load4<T>(reinterpret_cast<const T*>(vb) + page * p.v.sb + row * p.v.sl + v * 128 * p.v.sd, p.v.sd, p.wide_kv);
            }
          }
          for (row += kKeys; row >= p.page;) row -= p.page;
        }
        float x[kVals];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int s = 0; s < kAhead; ++s) {
            float z = 0.f;
#pragma unroll
            for (int v = 0; v < kVecs; ++v)
              z = fmaf(q[r][v].x, kx[s][v].x, fmaf(q[r][v].y, kx[s][v].y, fmaf(q[r][v].z, kx[s][v].z, fmaf(q[r][v].w, kx[s][v].w, z))));
            x[r * kAhead + s] = z;
          }
        lane_sums<kVals, kLanes / 2>(x, sub);  // score sub * kVals / kLanes and following ones
        const int first = sub * kVals / kLanes % kAhead;  // step of its first score
        float top = my_m;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int s = first + i;
          const bool is = ((there >> s) & (seen >> ((s0 + s) * kKeys + group)) & 1u) != 0;
          x[i] = is ? x[i] * p.scale_log2 : -CUDART_INF_F;
          top = fmaxf(top, x[i]);
        }
#pragma unroll
        for (int d = kRowLanes / 2; d >= kSame; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float safe = top == -CUDART_INF_F ? 0.f : top, a = tc::ex2(my_m - safe);
        my_m = top;
        my_l *= a;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int s = first + i;
          const bool is = ((there >> s) & (seen >> ((s0 + s) * kKeys + group)) & 1u) != 0;
          const float w = tc::ex2(x[i] - safe);
          my_l += w;
          if (sub % kSame == 0) reinterpret_cast<float*>(weights[warp][group])[sub * kVals / kLanes + i] = is ? w : -1.f;
        }
        if (sub % kRowLanes == 0) alpha[warp][group][my_r] = a;
        const bool moved = __any_sync(0xffffffffu, a != 1.f);
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (moved) {
            const float ar = alpha[warp][group][r];
#pragma unroll
            for (int v = 0; v < kVecs; ++v) o[r][v].x *= ar, o[r][v].y *= ar, o[r][v].z *= ar, o[r][v].w *= ar;
          }
#pragma unroll
          for (int s4 = 0; s4 < kAhead; s4 += 4) {
            const float4 w4 = weights[warp][group][(r * kAhead + s4) / 4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float w = u == 0 ? w4.x : (u == 1 ? w4.y : (u == 2 ? w4.z : w4.w));
              if (!(w < 0.f)) {  // a hidden key may hold anything; what a visible one holds counts whatever its weight
#pragma unroll
                for (int v = 0; v < kVecs; ++v) {
                  o[r][v].x = fmaf(w, vx[s4 + u][v].x, o[r][v].x); o[r][v].y = fmaf(w, vx[s4 + u][v].y, o[r][v].y);
                  o[r][v].z = fmaf(w, vx[s4 + u][v].z, o[r][v].z); o[r][v].w = fmaf(w, vx[s4 + u][v].w, o[r][v].w);
                }
              }
            }
          }
        }
        __syncwarp();  // the weights have been read
      }
    }

    float m[R], l[R];
#pragma unroll
    for (int d = kRowLanes / 2; d >= kSame; d >>= 1) my_l += __shfl_xor_sync(0xffffffffu, my_l, d);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = __shfl_sync(0xffffffffu, my_m, group * kLanes + r * kRowLanes);
      l[r] = __shfl_sync(0xffffffffu, my_l, group * kLanes + r * kRowLanes);
    }
    // the groups' states, then the warps', become one
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int d = kLanes; d < 32; d <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m[r], d), l2 = __shfl_xor_sync(0xffffffffu, l[r], d), top = fmaxf(m[r], m2);
        const float safe = top == -CUDART_INF_F ? 0.f : top, a = exp2f(m[r] - safe), b = exp2f(m2 - safe);
        m[r] = top;
        l[r] = l[r] * a + l2 * b;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          o[r][v].x = o[r][v].x * a + __shfl_xor_sync(0xffffffffu, o[r][v].x, d) * b;
          o[r][v].y = o[r][v].y * a + __shfl_xor_sync(0xffffffffu, o[r][v].y, d) * b;
          o[r][v].z = o[r][v].z * a + __shfl_xor_sync(0xffffffffu, o[r][v].z, d) * b;
          o[r][v].w = o[r][v].w * a + __shfl_xor_sync(0xffffffffu, o[r][v].w, d) * b;
        }
      }
      if (group == 0) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) sums[warp][r][ch / 4 + v * 32] = o[r][v];
      }
      if (lane == 0) stat[warp][r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    for (int idx = tid; idx < R * (DP / 4); idx += WARPS * 32) {
      const int r = idx / (DP / 4), d = (idx % (DP / 4)) * 4;
      if (d >= p.D || t.r0 + r >= p.N * p.G) continue;
      float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, stat[w][r].x);
      float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
      const float safe = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float a = exp2f(stat[w][r].x - safe);
        const float4 y = sums[w][r][d / 4];
        sum = fmaf(a, stat[w][r].y, sum);
        z.x = fmaf(a, y.x, z.x); z.y = fmaf(a, y.y, z.y); z.z = fmaf(a, y.z, z.z); z.w = fmaf(a, y.w, z.w);
      }
      if (piece.slot < 0) {
        const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
        const float inv = r < rows && sum != 0.f ? 1.f / sum : 0.f;
        store4<T>(p, o_row<T>(p, t.b, h, i), d, z.x * inv, z.y * inv, z.z * inv, z.w * inv);
        if (d == 0) store_lse(p, t.b, h, i, r < rows, top, sum);
      } else {
        const long long at = (long long)piece.slot * p.rows + r;
        *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = z;
        if (d == 0) p.part_ml[at] = make_float2(top, sum);
      }
    }
  }
}

}  // namespace cache
}  // namespace chill
