// What the kernels of the paged cache share: geometry of a call, how the work is cut into equal shares, what a new token may see.
//
// Attention of new tokens over a cache, one (request, kv head) at a time: its rows are the new tokens times the heads that share
// the kv head, row r = token r / G, head r % G, in tiles of `rows` rows; its keys are the cached ones and the new ones, in tiles
// of kKeyTile keys.  A "unit" is one tile of rows of one kv head with the tiles of keys that it can see; units are numbered
// by request, tile of rows, kv head.  Lengths live on the GPU, so the host can not split long units: every CTA works out
// the prefix sum over the units' tiles and takes an equal share of all of them, wherever it begins and ends (in the middle of
// units, mostly).  What a CTA has of a unit that it does not cover alone goes to a workspace as (maximum, sum, un-normalised O), and
// a second kernel, launched behind the first without a gap, joins the parts in order of the keys: results are the same each run.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "generic.cuh"

namespace chill {
namespace cache {

constexpr int kMaxLen = 1 << 29;    // positions; three of them added stay below 2^31
constexpr int kKeyTile = 64;        // keys of a tile, in all kernels
constexpr int kScanEntries = 1024;  // (request, tile of rows) pairs whose prefix sum every CTA works out by itself

CHILL_HD int clamp_len(int x) { return imin(imax(x, 0), kMaxLen); }

struct CachedP {
  int B, H, Hkv, G, N, D;
  int page, num_pages, width;
  int box;              // rows of a TMA box (tensor-core kernels)
  bool wide_q, wide_o;  // rows of Q / O can be moved in 16-byte vectors
  int rows, row_tiles;  // rows of a tile, tiles of N * G rows
  int words;            // 32-bit words of an ancestor row
  int min_share;        // tiles of keys a CTA takes at least
  float scale_log2;     // softmax scale * log2(e)
  MaskArgs margs;
  TRef q, o;            // [batch][head][token][channel]
  TRef k, v;            // [page][head][row][channel]
  float* lse;           // may be null
  long long lse_sb, lse_sh, lse_sl;
  const int* table;
  long long table_sb;
  const int *lens, *new_lens;
  const int *positions, *ancestors;  // ancestors null: the new tokens are a chain
  // workspace
  const int* cum;       // prefix sums of a launch of their own; null: every CTA works them out
  int4* seam;           // [CTA]: the unit its share begins in: (entry, kv head, first tile, tiles)
  int* all;             // number of all tiles
  float2* part_ml;      // [2 * CTA + (0 first, 1 last unit of its share)][row]
  float* part_o;        // the same, [D]
  int* status;
};

// A tile of rows of one request: what it can see.
struct RowTile {
  int b, r0;
  int cached, fresh;  // tokens in the cache, new tokens
  int total;          // keys there are: cached + fresh, or what the table has room for
  int rows;           // valid rows from r0 on
  int p0, p1;         // positions of the rows, first and last (a hull for trees)
  int k_lo, n_tiles;  // first key (a multiple of kKeyTile) and tiles of keys; no tile: nothing is visible
  int full_lo, full_hi;  // keys that every row sees, half-open
};

template <class M>
__device__ __forceinline__ RowTile row_tile(const CachedP& p, int entry) {
  RowTile t;
  t.b = entry / p.row_tiles;
  t.r0 = (entry - t.b * p.row_tiles) * p.rows;
  t.cached = clamp_len(p.lens[t.b]);
  t.fresh = imin(imax(p.new_lens[t.b], 0), p.N);
  const int n = t.cached + t.fresh;
  t.total = imin(n, p.width * p.page);
  t.rows = imin(imax(t.fresh * p.G - t.r0, 0), p.rows);
  t.k_lo = t.n_tiles = t.full_lo = t.full_hi = 0;
  t.p0 = t.p1 = t.cached;
  if (t.rows == 0) return t;
  const bool tree = p.ancestors != nullptr;
  const int i0 = t.r0 / p.G, i1 = (t.r0 + t.rows - 1) / p.G;
  t.p0 = t.cached + (tree ? 0 : i0);
  t.p1 = t.cached + i1;  // a token of a tree is at most as deep as there are tokens before it
  int lo, hi;
  tile_range<M, true>(t.p0, t.p1 - t.p0 + 1, n, p.margs, lo, hi);
  if (tree) {  // cached keys by the mask, then the new ones up to the last row's own
    lo = hi >= lo ? imin(lo, t.cached) : t.cached;
    hi = t.p1;
  }
  lo = imax(lo, 0);
  hi = imin(hi, t.total - 1);
  if (hi < lo) return t;
  t.k_lo = lo / kKeyTile * kKeyTile;
  t.n_tiles = (hi - t.k_lo) / kKeyTile + 1;
  if (M::kHasKFullRange) {
    M::k_full_range_for_q(t.p0, t.p1 - t.p0 + 1, n, p.margs, t.full_lo, t.full_hi);
    t.full_hi = imin(t.full_hi, tree ? imin(t.cached, t.total) : t.total);
  }
  return t;
}

// Tiles a unit counts for in the shares: one at least, so that every unit has a CTA that writes its rows.
template <class M>
__device__ __forceinline__ int unit_tiles(const CachedP& p, int entry) {
  return imax(row_tile<M>(p, entry).n_tiles, 1);
}

// Position of row r (token i) of a tile, and whether it sees key t (a place in the cache), t < total.
__device__ __forceinline__ int token_position(const CachedP& p, const RowTile& t, int i) {
  return p.ancestors != nullptr ? p.positions[(long long)t.b * p.N + i] : t.cached + i;
}
template <class M>
__device__ __forceinline__ bool sees(const CachedP& p, const RowTile& t, int i, int pos, int key) {
  const int n = t.cached + t.fresh;
  if (key < t.cached || p.ancestors == nullptr) return M::mask(pos, key, n, p.margs);
  const int j = key - t.cached;
  const unsigned word = (unsigned)p.ancestors[((long long)t.b * p.N + i) * p.words + (j >> 5)];
  return ((word >> (j & 31)) & 1u) != 0 && M::mask(pos, p.positions[(long long)t.b * p.N + j], n, p.margs);
}

// cum[e] = tiles of the (request, tile of rows) pairs before e, of one kv head; e <= B * row_tiles.  THREADS threads.
template <class M, int THREADS>
__device__ __forceinline__ void scan_units(const CachedP& p, int entries, int* cum) {
  __shared__ int sums[THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int carry = 0;
  for (int base = 0; base < entries; base += THREADS) {
    const int e = base + (int)threadIdx.x;
    const int v = e < entries ? unit_tiles<M>(p, e) : 0;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      const int s = sums[w];
      if (w < warp) before += s;
      carry += s;
    }
    if (e < entries) cum[e] = before + x - v;
    __syncthreads();
  }
  if (threadIdx.x == 0) cum[entries] = carry;
  __syncthreads();
}

template <class M>
__global__ void __launch_bounds__(1024) scan_kernel(CachedP p, int* cum) {
  scan_units<M, 1024>(p, p.B * p.row_tiles, cum);
}

// The share of CTA c of `ctas`: tiles [first, last) of all Hkv * cum[entries].  With little work only as many CTAs take part as
// have min_share tiles each.
__device__ __forceinline__ int share_begin(int total, int ctas, int c) { return (int)((long long)total * c / ctas); }
__device__ __forceinline__ int active_ctas(const CachedP& p, int total, int grid) {
  return imin(grid, imax(1, total / p.min_share));
}
// The entry whose tiles (of all kv heads) hold tile t.
__device__ __forceinline__ int find_entry(const int* cum, int entries, int hkv, int t) {
  int lo = 0, hi = entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cum[mid] * hkv <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A piece of a CTA's share: tiles [t0, t1) of the keys of one unit.
struct Piece {
  int entry, head;
  int t0, t1;
  bool whole;  // the unit is this CTA's alone
  int slot;    // of the workspace, when it is not
};

// Walks a CTA's share piece by piece; all threads of the CTA call it alike.
struct Share {
  int first, last, at, entry;
  __device__ __forceinline__ bool next(const CachedP& p, const int* cum, Piece& x) {
    if (at >= last) return false;
    while (cum[entry + 1] * p.Hkv <= at) ++entry;
    const int tiles = cum[entry + 1] - cum[entry], base = cum[entry] * p.Hkv;
    x.entry = entry;
    x.head = (at - base) / tiles;
    const int begin = base + x.head * tiles;
    x.t0 = at - begin;
    x.t1 = imin(last - begin, tiles);
    x.whole = x.t0 == 0 && x.t1 == tiles;
    x.slot = 2 * (int)blockIdx.x + (at == first ? 0 : 1);
    at = begin + x.t1;
    return true;
  }
};

// Prefix sums, this CTA's share and, for the kernel that joins the parts, where the share begins.
template <class M, int THREADS>
__device__ __forceinline__ Share begin_share(const CachedP& p, int* smem_cum, const int*& cum) {
  const int entries = p.B * p.row_tiles;
  cum = p.cum;
  if (cum == nullptr) {
    scan_units<M, THREADS>(p, entries, smem_cum);
    cum = smem_cum;
  }
  const int total = cum[entries] * p.Hkv, ctas = active_ctas(p, total, (int)gridDim.x), c = (int)blockIdx.x;
  Share s;
  s.first = c < ctas ? share_begin(total, ctas, c) : total;
  s.last = c < ctas ? share_begin(total, ctas, c + 1) : total;
  s.at = s.first;
  s.entry = s.first < s.last ? find_entry(cum, entries, p.Hkv, s.first) : 0;
  if (threadIdx.x == 0) {
    int4 seam = make_int4(0, 0, 0, 0);
    if (s.first < s.last) {
      const int tiles = cum[s.entry + 1] - cum[s.entry], head = (s.first - cum[s.entry] * p.Hkv) / tiles;
      seam = make_int4(s.entry, head, cum[s.entry] * p.Hkv + head * tiles, tiles);
    }
    p.seam[c] = seam;
    if (c == 0) *p.all = total;
  }
  return s;
}

// One tile of 64 keys by TMA: lane i of a warp copies box i % boxes.  The page of box i of the tile at k0; without one, page
// num_pages, which is outside the map: TMA fills the box with zeros.
__device__ __forceinline__ int tile_page(const CachedP& p, const RowTile& t, int k0, int i, bool& there) {
  const int at = k0 + i * p.box;
  int page = -1;
  if (at < t.total) page = p.table[t.b * p.table_sb + at / p.page];
  there = page >= 0 && page < p.num_pages;
  return there ? page : p.num_pages;
}
// Groups of 8 keys without a page, from the boxes without one.
__device__ __forceinline__ int lost_groups(const CachedP& p, unsigned lost, int boxes) {
  int groups = 0;
  if (lost != 0)
    for (int i = 0; i < boxes; ++i)
      if ((lost >> i) & 1u) groups |= ((1 << (p.box / 8)) - 1) << (i * (p.box / 8));
  return groups;
}

__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Writes one element of O and, by whoever has channel 0, the LSE.
template <typename T>
__device__ __forceinline__ T* o_row(const CachedP& p, int b, int h, int i) {
  return reinterpret_cast<T*>(p.o.p) + b * p.o.sb + h * p.o.sh + i * p.o.sl;
}
__device__ __forceinline__ void store_lse(const CachedP& p, int b, int h, int i, bool valid, float m, float l) {
  if (p.lse == nullptr) return;
  float x = 0.f;
  if (valid) x = l == 0.f ? -CUDART_INF_F : m + log2f(l);
  p.lse[b * p.lse_sb + h * p.lse_sh + i * p.lse_sl] = x;
}

// ------------------------------------------------------------------------------------------------------- joining
// Block (c, y): the unit that the boundary between the shares of CTAs c and c + 1 cuts, if that is the first boundary inside it;
// rows y * rows / gridDim.y on.  O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over the parts in order.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(CachedP p, int grid) {
  pdl_wait();
  const int c = (int)blockIdx.x + 1;
  const int total = *p.all, ctas = active_ctas(p, total, grid);
  if (c >= ctas) return;
  const int4 u = p.seam[c];
  const int cut = share_begin(total, ctas, c), before = share_begin(total, ctas, c - 1);
  if (cut == u.z || before > u.z) return;  // a unit begins here; or an earlier block joins this one
  const int end = u.z + u.w;
  const int slot0 = 2 * (c - 1) + (before < u.z ? 1 : 0);
  int parts = 2;  // CTAs c - 1, c, ... as long as their shares begin inside the unit
  while (c - 1 + parts < ctas && share_begin(total, ctas, c - 1 + parts) < end) ++parts;

  const int b = u.x / p.row_tiles, r0 = (u.x - b * p.row_tiles) * p.rows;
  const int all = p.N * p.G, valid = imin(imax(p.new_lens[b], 0), p.N) * p.G;
  const int per_row = p.D / 4, chunk = p.rows / (int)gridDim.y, from = (int)blockIdx.y * chunk;
  for (int idx = threadIdx.x; idx < chunk * per_row; idx += 256) {
    const int r = from + idx / per_row, d = (idx % per_row) * 4;
    if (r0 + r >= all) break;
    const int i = (r0 + r) / p.G, h = u.y * p.G + (r0 + r) % p.G;
    const bool ok = r0 + r < valid;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ok) {
      for (int k = 0; k < parts; ++k) m = fmaxf(m, p.part_ml[(long long)(k == 0 ? slot0 : 2 * (c - 1 + k)) * p.rows + r].x);
      if (m != -CUDART_INF_F) {
        for (int k = 0; k < parts; ++k) {
          const long long at = (long long)(k == 0 ? slot0 : 2 * (c - 1 + k)) * p.rows + r;
          const float2 ml = p.part_ml[at];
          const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * p.D + d);
          const float w = exp2f(ml.x - m);
          l += w * ml.y;
          o.x += w * x.x; o.y += w * x.y; o.z += w * x.z; o.w += w * x.w;
        }
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    }
    T* to = o_row<T>(p, b, h, i);
    to[d * p.o.sd] = from_f<T>(o.x); to[(d + 1) * p.o.sd] = from_f<T>(o.y);
    to[(d + 2) * p.o.sd] = from_f<T>(o.z); to[(d + 3) * p.o.sd] = from_f<T>(o.w);
    if (d == 0) store_lse(p, b, h, i, ok, m, l);
  }
}

}  // namespace cache
}  // namespace chill
