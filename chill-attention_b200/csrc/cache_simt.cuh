// Attention of new tokens over a paged cache on the CUDA cores: fp32 (IEEE arithmetic) and every layout that the tensor-core
// kernels can not take.  See cache_common.cuh for units and shares.
//
// Up to 8 rows (simt_few): bound by memory, so nothing goes through shared memory.  D / 4 lanes (32 at most) share a key, a warp has
// 16 keys of every tile of 64; a lane keeps four channels (eight at head dim 256) of Q and O of every row, reads those of K and V of
// four or eight steps at once, and gets the scores by butterflies over its lanes.  Every group of lanes has a maximum and a sum of its own: no warp,
// and no group, waits for another before the end of a piece.
//
// More rows: a CTA of 128 threads works on 16 rows and 64 keys at a time, everything as fp32 in shared memory:
//   S = Q K^T   a thread has one key and 8 rows: one vector of K and 8 (broadcast) of Q for 32 FMAs
//   softmax     a warp has 4 rows; running maximum and sum in base 2
//   O += P V    a thread has 4 channels of 2 D / 64 rows (registers)
#pragma once
#include "cache_common.cuh"
#include "tc_common.cuh"

namespace chill {
namespace cache {

constexpr int kSimtThreads = 128;
constexpr int kSimtRows = 16;

template <int DP>
struct SimtSmem {
  static constexpr int kKRow = DP + 4;  // floats of a K row: 16-byte vectors of 8 consecutive keys fall into different banks
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kSimtRows * DP;
  static constexpr int kV = kK + kKeyTile * kKRow;
  static constexpr int kS = kV + kKeyTile * DP;
  static constexpr int kM = kS + kSimtRows * kKeyTile;  // alpha of every row
  static constexpr int kBad = kM + kSimtRows;           // a key has no page
  static constexpr int kItem = kBad + kKeyTile;
  static constexpr int kCum = kItem + (int)sizeof(Item) / 4;
  static constexpr int kBytes = (kCum + kScanEntries + 1) * 4;
};

template <typename T, int DP, class M>
__global__ void __launch_bounds__(kSimtThreads) cached_simt_kernel(const __grid_constant__ CachedP p) {
  using L = SimtSmem<DP>;
  extern __shared__ __align__(16) float smem[];
  float *sq = smem + L::kQ, *sk = smem + L::kK, *sv = smem + L::kV, *ss = smem + L::kS, *sa = smem + L::kM;
  int* bad = reinterpret_cast<int*>(smem + L::kBad);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kChunks = DP / 4;                                                   // channel quads
  constexpr int kGroups = kSimtThreads / kChunks < kSimtRows ? kSimtThreads / kChunks : kSimtRows;  // threads of a quad
  constexpr int kOwn = kSimtRows / kGroups;                                         // rows of a thread in O += P V
  const int quad = tid % kChunks, group = tid / kChunks;
  const bool pv = group < kGroups;
  Item& item = *reinterpret_cast<Item*>(smem + L::kItem);
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
    const int tiles = item.tiles;
    for (int idx = tid; idx < kSimtRows * DP; idx += kSimtThreads) {
      const int r = idx / DP, d = idx % DP;
      float x = 0.f;
      if (r < t.rows && d < p.D) {
        const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
        x = to_f(row_ptr<T>(p.q, t.b, h, i)[d * p.q.sd]);
      }
      sq[r * DP + d] = x;
    }
    float m[4], l[4];  // rows 4 * warp + n, the same in all lanes
    float acc[kOwn][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) m[n] = -CUDART_INF_F, l[n] = 0.f;
#pragma unroll
    for (int n = 0; n < kOwn; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    for (int kt = piece.t0; kt < tiles; ++kt) {
      const int k0 = t.k_lo + kt * kKeyTile;
      __syncthreads();  // the tile before has been used
      for (int idx = tid; idx < kKeyTile * kChunks; idx += kSimtThreads) {
        const int key = idx / kChunks, d = (idx % kChunks) * 4, at = k0 + key;
        const int page = at < t.total ? p.table[t.b * p.table_sb + at / p.page] : -1;
        const bool there = page >= 0 && page < p.num_pages;
        float4 kx = make_float4(0.f, 0.f, 0.f, 0.f), vx = kx;
        if (there) {
          const int row = at % p.page;
          const T* ks = reinterpret_cast<const T*>(p.k.p) + page * p.k.sb + piece.head * p.k.sh + row * p.k.sl;
          const T* vs = reinterpret_cast<const T*>(p.v.p) + page * p.v.sb + piece.head * p.v.sh + row * p.v.sl;
          float* kf = &kx.x;
          float* vf = &vx.x;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (d + u < p.D) {
              kf[u] = to_f(ks[(d + u) * p.k.sd]);
              vf[u] = to_f(vs[(d + u) * p.v.sd]);
            }
          }
        }
        *reinterpret_cast<float4*>(sk + key * L::kKRow + d) = kx;
        *reinterpret_cast<float4*>(sv + key * DP + d) = vx;
        if (d == 0) bad[key] = !there;
      }
      __syncthreads();
      {  // S: key tid % 64, rows 8 * (tid / 64) on
        const int key = tid & 63, r0 = (tid >> 6) * 8;
        float s[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = 0.f;
#pragma unroll 4
        for (int d = 0; d < DP; d += 4) {
          const float4 kx = *reinterpret_cast<const float4*>(sk + key * L::kKRow + d);
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const float4 qx = *reinterpret_cast<const float4*>(sq + (r0 + n) * DP + d);
            s[n] = fmaf(qx.x, kx.x, fmaf(qx.y, kx.y, fmaf(qx.z, kx.z, fmaf(qx.w, kx.w, s[n]))));
          }
        }
        const int at = k0 + key;
        const bool full = at >= t.full_lo && at < t.full_hi;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const int r = r0 + n;
          bool ok = r < t.rows && at < t.total && !bad[key];
          if (ok && !full) {
            const int i = (t.r0 + r) / p.G;
            ok = sees<M>(p, t, i, token_position(p, t, i), at);
          }
          ss[r * kKeyTile + key] = ok ? s[n] * p.scale_log2 : -CUDART_INF_F;
        }
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < 4; ++n) {  // softmax of row 4 * warp + n
        float* row = ss + (warp * 4 + n) * kKeyTile;
        const float x = row[lane], y = row[lane + 32];
        float top = fmaxf(x, y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m[n], top), safe = m_new == -CUDART_INF_F ? 0.f : m_new;
        const float a = exp2f(m[n] - safe);  // m = -inf: 0
        const float ex = exp2f(x - safe), ey = exp2f(y - safe);
        l[n] = l[n] * a + warp_sum(ex + ey);
        m[n] = m_new;
        row[lane] = ex;
        row[lane + 32] = ey;
        if (lane == 0) sa[warp * 4 + n] = a;
      }
      __syncthreads();
      if (pv) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
          const float a = sa[group * kOwn + n];
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[n][u] *= a;
        }
#pragma unroll 4
        for (int key = 0; key < kKeyTile; ++key) {
          const float4 vx = *reinterpret_cast<const float4*>(sv + key * DP + quad * 4);
#pragma unroll
          for (int n = 0; n < kOwn; ++n) {
            const float w = ss[(group * kOwn + n) * kKeyTile + key];
            if (w != 0.f) {  // a hidden key may hold anything
              acc[n][0] = fmaf(w, vx.x, acc[n][0]); acc[n][1] = fmaf(w, vx.y, acc[n][1]);
              acc[n][2] = fmaf(w, vx.z, acc[n][2]); acc[n][3] = fmaf(w, vx.w, acc[n][3]);
            }
          }
        }
      }
    }

    // maximum and sum of every row, for the threads that hold its O
    __syncthreads();
    float* sm = ss;
    if (lane < 4) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (lane == n) sm[warp * 4 + n] = m[n], sm[kSimtRows + warp * 4 + n] = l[n];
    }
    __syncthreads();
    if (pv) {
#pragma unroll
      for (int n = 0; n < kOwn; ++n) {
        const int r = group * kOwn + n, all = p.N * p.G;
        if (t.r0 + r >= all) continue;
        const float mr = sm[r], lr = sm[kSimtRows + r];
        if (piece.slot < 0) {
          const int i = (t.r0 + r) / p.G, h = piece.head * p.G + (t.r0 + r) % p.G;
          const float inv = r < t.rows && lr > 0.f ? 1.f / lr : 0.f;
          T* to = o_row<T>(p, t.b, h, i);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (quad * 4 + u < p.D) to[(quad * 4 + u) * p.o.sd] = from_f<T>(acc[n][u] * inv);
          if (quad == 0) store_lse(p, t.b, h, i, r < t.rows, mr, lr);
        } else {
          const long long at = (long long)piece.slot * p.rows + r;
          if (quad * 4 < p.D) *reinterpret_cast<float4*>(p.part_o + at * p.D + quad * 4) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
          if (quad == 0) p.part_ml[at] = make_float2(mr, lr);
        }
      }
    }
  }
}

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

// WARPS: four of them have a tile; with eight (units taken whole, where one CTA has all of a unit's tiles) two tiles are under way.
template <typename T, int DP, int R, int WARPS, class M>
__global__ void __launch_bounds__(WARPS * 32) cached_simt_few_kernel(const __grid_constant__ CachedP p) {
  constexpr int kLanes = DP / 4 < 32 ? DP / 4 : 32;     // of a key
  constexpr int kVecs = DP / 4 / kLanes;                // vectors of four channels of a lane
  constexpr int kKeys = 32 / kLanes;                    // keys of a warp at a time: its groups of lanes
  constexpr int kSteps = 16 / kKeys;                    // of the warp's 16 keys of a tile
  constexpr int kAhead = kSteps < (R == 4 ? 8 / kVecs : 4) ? kSteps : (R == 4 ? 8 / kVecs : 4);  // steps whose loads are in flight
  __shared__ float4 sums[WARPS][R][DP / 4];
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
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -CUDART_INF_F;
      l[r] = 0.f;
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
    for (int kt = piece.t0 + warp / 4; kt < tiles; kt += WARPS / 4) {
      const int k0 = k_lo + kt * kKeyTile + quarter;
      if (k0 >= total) break;
      unsigned seen = rows >= 32 ? 0xffffffffu : (1u << rows) - 1u, words[R];  // bit s * kKeys + g: the key of group g in step s
      if (k0 < full_lo || k0 + 16 > full_hi) {
        const uint64_t vis = visible_keys<M>(p, t, my_token, my_pos, my_near, k0 - quarter, 0);
        __syncwarp();
        seen = (unsigned)(vis >> quarter) & 0xffffu;  // row `lane`'s 16 keys of this warp
#pragma unroll
        for (int r = 0; r < R; ++r) words[r] = __shfl_sync(0xffffffffu, seen, r);
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) words[r] = (seen >> r) & 1u ? 0xffffu : 0u;
      }
#pragma unroll 1
      for (int s0 = 0; s0 < kSteps; s0 += kAhead) {
        float4 kx[kAhead][kVecs], vx[kAhead][kVecs];
        unsigned there = 0;
        int key = k0 + s0 * kKeys + group, block = key / p.page, row = key - block * p.page;
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
          const int page = key < total ? table[block] : -1;
          const bool is = page >= 0 && page < p.num_pages;
          there |= (unsigned)is << s;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            kx[s][v] = vx[s][v] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (is && ch + v * 128 < p.D) {
              kx[s][v] = load4<T>(reinterpret_cast<const T*>(kb) + page * p.k.sb + row * p.k.sl + v * 128 * p.k.sd, p.k.sd, p.wide_kv);
              vx[s][v] = load4<T>(reinterpret_cast<const T*>(vb) + page * p.v.sb + row * p.v.sl + v * 128 * p.v.sd, p.v.sd, p.wide_kv);
            }
          }
          key += kKeys;
          for (row += kKeys; row >= p.page; row -= p.page) ++block;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float x[kAhead], top = m[r];
#pragma unroll
          for (int s = 0; s < kAhead; ++s) {
            x[s] = 0.f;
#pragma unroll
            for (int v = 0; v < kVecs; ++v)
              x[s] = fmaf(q[r][v].x, kx[s][v].x, fmaf(q[r][v].y, kx[s][v].y, fmaf(q[r][v].z, kx[s][v].z, fmaf(q[r][v].w, kx[s][v].w, x[s]))));
          }
#pragma unroll
          for (int d = kLanes / 2; d > 0; d >>= 1)
#pragma unroll
            for (int s = 0; s < kAhead; ++s) x[s] += __shfl_xor_sync(0xffffffffu, x[s], d);
          unsigned see = 0;  // the same in all lanes of a group
#pragma unroll
          for (int s = 0; s < kAhead; ++s) {
            const bool is = ((there >> s) & (words[r] >> ((s0 + s) * kKeys + group)) & 1u) != 0;
            see |= (unsigned)is << s;
            x[s] = is ? x[s] * p.scale_log2 : -CUDART_INF_F;
            top = fmaxf(top, x[s]);
          }
          const float safe = top == -CUDART_INF_F ? 0.f : top, a = tc::ex2(m[r] - safe);
          m[r] = top;
          l[r] *= a;
#pragma unroll
          for (int v = 0; v < kVecs; ++v) o[r][v].x *= a, o[r][v].y *= a, o[r][v].z *= a, o[r][v].w *= a;
#pragma unroll
          for (int s = 0; s < kAhead; ++s) {
            if ((see >> s) & 1u) {  // a hidden key may hold anything
              const float w = tc::ex2(x[s] - safe);
              l[r] += w;
#pragma unroll
              for (int v = 0; v < kVecs; ++v) {
                o[r][v].x = fmaf(w, vx[s][v].x, o[r][v].x); o[r][v].y = fmaf(w, vx[s][v].y, o[r][v].y);
                o[r][v].z = fmaf(w, vx[s][v].z, o[r][v].z); o[r][v].w = fmaf(w, vx[s][v].w, o[r][v].w);
              }
            }
          }
        }
      }
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
