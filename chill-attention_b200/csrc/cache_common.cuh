// What the kernels of the paged cache share: geometry of a call, how the work is cut into shares, what a new token may see, how parts
// are joined.
//
// Attention of new tokens over a cache, one (request, kv head) at a time: its rows are the new tokens times the heads that share
// the kv head, row r = token r / G, head r % G, in tiles of `rows` rows; its keys are the cached ones and the new ones, in tiles
// of kKeyTile keys.  A "unit" is one tile of rows of one kv head with the tiles of keys that it can see; units are numbered
// by request, tile of rows, kv head.  Lengths live on the GPU, so the host can not split long units: every CTA sums up the units' tiles
// (with very many units a kernel of its own does) and cuts all of them into the same shares, wherever these begin and end (in the middle
// of units, mostly).  Every CTA has one large share; where the kernel is bound by memory the last sixth of the tiles is cut into small
// shares that go to whoever is done first, because SMs get unequal parts of the bandwidth (equal shares of 160 us were done after
// 143 to 184 us).
// What a share has of a unit that it does not cover alone goes to a workspace as (maximum, sum, un-normalised O), and a kernel launched
// behind joins the parts in order of the keys: results are the same each run, whichever CTA had which share.  (Joined by the CTA of the last
// part instead, a unit of 16 rows in 148 parts kept one CTA busy for 80 us, and the fence that takes cost every piece 3 us.  A first kernel
// that plans for all CTAs takes 6 us, this sum 2 us.)
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "generic.cuh"

namespace chill {
namespace cache {

constexpr int kMaxLen = 1 << 29;    // positions; three of them added stay below 2^31
constexpr int kKeyTile = 64;        // keys of a tile, in all kernels
constexpr int kTileRows = 128;      // rows of a tile of the kernel for many rows, at most
constexpr int kTailFrom = 24;       // tiles a CTA, from where on there are small shares
constexpr int kTailTiles = 8;       // tiles of a small share, at least
constexpr int kScanEntries = 256;   // (request, tile of rows) pairs that every CTA sums up by itself
constexpr int kScanThreads = 1024;

// CTAs on an SM of the kernel for few rows with D channels and `rows` rows a tile.  Small tiles take a CTA mostly latency: 64 requests, one
// token each, head dim 64: 120 us with two, 110 with three.
__host__ __device__ constexpr int rows_ctas(int D, int rows) { return D > 128 ? 1 : (D <= 64 && rows == 16 ? 3 : 2); }

CHILL_HD int clamp_len(int x) { return imin(imax(x, 0), kMaxLen); }

struct CachedP {
  int B, H, Hkv, G, N, D;
  int page, num_pages, width;
  int box;              // rows of a TMA box (tensor-core kernels)
  bool wide_q, wide_o;  // rows of Q / O can be moved in 16-byte vectors
  bool wide_kv;         // those of the caches too
  int rows, row_tiles;  // rows of a tile, tiles of N * G rows
  int words;            // 32-bit words of an ancestor row
  bool whole;           // short tables: CTAs take whole units in turn, nothing is summed up, cut or joined
  int pad;              // tiles that a unit counts for beside its own
  int min_share;        // tiles of keys of a share at least
  int tail_shares;      // small shares behind the large ones, at most (0: none)
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
  const int* cum;       // [entries + 1]: tiles of the entries before, of one kv head, by a kernel of its own; null: every CTA for itself
  int* queue;           // [1]: small shares taken
  struct Seam* seams;   // [share]: the unit that is cut at the share's end for the first time
  float2* part_ml;      // [2 * share + (0 first, 1 last unit of the share)][row]
  float* part_o;        // the same, [D]; of the kernel for many rows [D / 4][row][4]
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

// What a unit counts for in the shares: its tiles, one at least, so that every unit has a CTA that writes its rows; and ahead of
// them `pad` for what a CTA spends on a unit beside its tiles.
template <class M>
__device__ __forceinline__ int unit_tiles(const CachedP& p, int entry) {
  return imax(row_tile<M>(p, entry).n_tiles, 1) + p.pad;
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

__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------------- shares
// cum[e] = tiles of the entries before e, of one kv head; e <= entries.
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
      const int y = sums[w];
      if (w < warp) before += y;
      carry += y;
    }
    if (e < entries) cum[e] = before + x - v;
    __syncthreads();
  }
  if (threadIdx.x == 0) cum[entries] = carry;
  __syncthreads();
}

// How the tiles of all units are cut: `large` equal shares up to tile large_end, then small ones of `tail` tiles.
struct Cut {
  int total, large_end, large, tail, shares;
  int each, more;  // tiles of a large share; so many of them have one more
  __device__ __forceinline__ int begin(int x) const {
    return x < large ? x * each + imin(x, more) : imin(total, large_end + (x - large) * tail);
  }
  __device__ __forceinline__ int of(int t) const {  // the share that tile t is in
    if (t >= large_end) return large + (t - large_end) / tail;
    const int longer = more * (each + 1);
    return t < longer ? t / (each + 1) : more + (t - longer) / each;
  }
};
__device__ __forceinline__ Cut make_cut(const CachedP& p, int total, int grid) {
  Cut c;
  c.total = c.large_end = total;
  c.large = c.shares = imax(1, imin(grid, total / p.min_share));
  c.tail = 1;
  if (p.tail_shares > 0 && total >= kTailFrom * grid) {
    const int rest = total / 6;
    c.tail = imax(kTailTiles, (rest + p.tail_shares - 1) / p.tail_shares);
    c.large_end = total - rest;
    c.shares = c.large + (rest + c.tail - 1) / c.tail;
  }
  c.each = c.large_end / c.large;
  c.more = c.large_end - c.each * c.large;
  return c;
}

// Before the launch of the attention kernel, which it overlaps: the counter of small shares, and where there are many entries their sums.
template <class M>
__global__ void __launch_bounds__(kScanThreads) prepare_kernel(const __grid_constant__ CachedP p, int* cum) {
  pdl_launch_dependents();
  if (threadIdx.x == 0) *p.queue = 0;
  if (cum != nullptr) scan_units<M, kScanThreads>(p, p.B * p.row_tiles, cum);
}

// The parts of a unit that is cut: slot0 of the share it begins in, then slot 2 * share of the following ones.
struct Seam {
  int parts;  // 0: the share's last unit ends with it, or begins before it
  int slot0;
  int b, head, r0, rows;
};

// The sums and the cut, by all threads of a CTA of the attention kernel.
template <class M, int THREADS>
__device__ __forceinline__ Cut begin_work(const CachedP& p, int* smem_cum, const int*& cum) {
  const int entries = p.B * p.row_tiles;
  cum = p.cum;
  if (p.whole) {
    Cut units{};
    units.shares = entries * p.Hkv;
    return units;
  }
  if (cum == nullptr) {
    scan_units<M, THREADS>(p, entries, smem_cum);
    cum = smem_cum;
  } else {
    pdl_wait();
  }
  const Cut cut = make_cut(p, cum[entries] * p.Hkv, (int)gridDim.x);
  if (threadIdx.x == 0)  // shares that there are not have nothing to join
    for (int c = (int)blockIdx.x; c < (int)gridDim.x + p.tail_shares; c += (int)gridDim.x)
      if (c >= cut.shares) p.seams[c].parts = 0;
  return cut;
}

// A piece of a share: tiles [t0, t1) of the keys of one unit.
struct Piece {
  int entry, head;  // entry < 0: there is no more
  int t0, t1;
  int slot;         // of the workspace; -1: the unit is this share's alone
};
struct Item {
  RowTile t;
  Piece x;
  int tiles;  // t1, or 0 where nothing is visible
};
// Hands out the pieces of a CTA's large share, then of small ones; a warp walks it, all lanes alike.
struct Work {
  Cut cut;
  const int* cum;
  int share, ahead;  // ahead: the small share that comes next (lane 0)
  int at, last, begin, tiles, entry, head;
  int pieces;        // of the share so far
  Seam seam;
  template <class M>
  __device__ __forceinline__ void open(const CachedP& p, int c) {
    share = c;
    if (c >= cut.shares) return;
    pieces = 0;
    seam.parts = 0;
    at = cut.begin(c);
    last = cut.begin(c + 1);
    int lo = 0, hi = p.B * p.row_tiles - 1;  // the entry whose tiles, of all kv heads, hold the first tile
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum[mid] * p.Hkv <= at) lo = mid;
      else hi = mid - 1;
    }
    entry = lo;
    tiles = cum[lo + 1] - cum[lo];
    head = (at - cum[lo] * p.Hkv) / tiles;
    begin = cum[lo] * p.Hkv + head * tiles;
  }
  template <class M>
  __device__ __forceinline__ void start(const CachedP& p, const Cut& c, const int* sums) {
    cut = c;
    cum = sums;
    ahead = 0;
    share = (int)blockIdx.x;
    if (!p.whole) open<M>(p, (int)blockIdx.x < cut.large ? (int)blockIdx.x : cut.shares);
  }
  // The share has been handed out: what of it is to be joined, and which one comes next.
  __device__ __forceinline__ void close(const CachedP& p) {
    if ((threadIdx.x & 31) == 0) {
      p.seams[share] = seam;
      if (p.tail_shares > 0) pdl_wait();  // prepare_kernel has cleared the counter; also where nobody asks it, or the call could end before that kernel
      if (cut.shares > cut.large) ahead = cut.large + atomicAdd(p.queue, 1);
    }
    __syncwarp();
  }
  template <class M>
  __device__ __forceinline__ bool next(const CachedP& p, Item& it) {
    Piece& x = it.x;
    x.entry = -1;
    if (p.whole) {  // share: a unit
      if (share >= cut.shares) return false;
      x.entry = share / p.Hkv;
      x.head = share - x.entry * p.Hkv;
      x.t0 = 0;
      x.slot = -1;
      it.t = row_tile<M>(p, x.entry);
      x.t1 = it.tiles = it.t.n_tiles;
      share += (int)gridDim.x;
      return true;
    }
    while (true) {
      if (share < cut.shares && at >= last) open<M>(p, cut.shares > cut.large ? __shfl_sync(0xffffffffu, ahead, 0) : cut.shares);
      if (share >= cut.shares) return false;
      if (at >= begin + tiles) {  // the next unit
        begin += tiles;
        if (++head == p.Hkv) {
          head = 0;
          ++entry;
          tiles = cum[entry + 1] - cum[entry];
        }
      }
      at = imax(at, imin(begin + p.pad, last));
      if (at < last) break;
      close(p);
    }
    const int first = begin + p.pad, real = tiles - p.pad;  // the unit's tiles
    x.entry = entry;
    x.head = head;
    x.t0 = at - first;
    x.t1 = imin(last - first, real);
    it.t = row_tile<M>(p, entry);
    it.tiles = it.t.n_tiles == 0 ? 0 : x.t1;
    const bool goes_on = x.t1 != real;
    x.slot = x.t0 != 0 || goes_on ? 2 * share + (pieces > 0 ? 1 : 0) : -1;
    if (x.t0 == 0 && goes_on) {
      seam.parts = cut.of(first + real - 1) - share + 1;
      seam.slot0 = x.slot;
      seam.b = it.t.b; seam.head = head; seam.r0 = it.t.r0; seam.rows = it.t.rows;
    }
    ++pieces;
    at = first + x.t1;
    if (at >= last) close(p);
    return true;
  }
};

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

// The first 64 of token i's ancestor bits, loaded ahead of the tiles that need them.
__device__ __forceinline__ uint64_t first_ancestors(const CachedP& p, int b, int i) {
  if (p.ancestors == nullptr || i < 0) return 0ull;
  const int* row = p.ancestors + ((long long)b * p.N + i) * p.words;
  return (uint64_t)(unsigned)row[0] | (p.words > 1 ? (uint64_t)(unsigned)row[1] << 32 : 0ull);
}

// Keys k0 .. k0 + 63 that token i at position pos sees, as bits; `near`: first_ancestors; `lost`: groups of 8 keys without a page.
template <class M>
__device__ __forceinline__ uint64_t visible_keys(const CachedP& p, const RowTile& t, int i, int pos, uint64_t near, int k0, int lost) {
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
    const int j0 = k0 - t.cached;  // number of the new token at the tile's first key
    uint64_t bits;
    if (p.words <= 2) {
      bits = j0 >= 64 ? 0ull : (j0 >= 0 ? near >> j0 : near << -j0);
    } else {
      const int* row = p.ancestors + ((long long)t.b * p.N + i) * p.words;
      const int w = imax(j0, 0) >> 5, sh = imax(j0, 0) & 31;
      auto word = [&](int x) -> uint64_t { return x < p.words ? (uint64_t)(unsigned)row[x] : 0ull; };
      bits = (word(w) | (word(w + 1) << 32)) >> sh;
      if (sh != 0) bits |= word(w + 2) << (64 - sh);
      if (j0 < 0) bits <<= -j0;
    }
    bits &= below(there);
    // ancestors stand at positions [cached, pos]: one look where the mask shows the token all of these
    int lo = 0, hi = 0;
    if (M::kHasKFullRange) M::k_full_range_for_q(pos, 1, n, p.margs, lo, hi);
    if (lo > t.cached || hi <= pos) {
      const int* at = p.positions + (long long)t.b * p.N + j0;
      for (uint64_t left = bits; left != 0ull;) {
        const int c = __ffsll((long long)left) - 1;
        left &= left - 1ull;
        if (!M::mask(pos, at[c], n, p.margs)) bits &= ~(1ull << c);
      }
    }
    vis |= bits;
  }
  for (int g = lost; g != 0; g &= g - 1) vis &= ~(0xffull << (8 * (__ffs(g) - 1)));
  return vis;
}

// Four channels of a row of O.
template <typename T>
__device__ __forceinline__ void store4(const CachedP& p, T* row, int ch, float a, float b, float c, float d) {
  if (p.wide_o) {  // channels side by side, rows on 16-byte boundaries
    if constexpr (sizeof(T) == 2) {
      T e[4] = {from_f<T>(a), from_f<T>(b), from_f<T>(c), from_f<T>(d)};
      *reinterpret_cast<uint2*>(row + ch) = *reinterpret_cast<const uint2*>(e);
    } else {
      *reinterpret_cast<float4*>(row + ch) = make_float4(a, b, c, d);
    }
  } else {
    row[ch * p.o.sd] = from_f<T>(a); row[(ch + 1) * p.o.sd] = from_f<T>(b);
    row[(ch + 2) * p.o.sd] = from_f<T>(c); row[(ch + 3) * p.o.sd] = from_f<T>(d);
  }
}

// ------------------------------------------------------------------------------------------------------- joining
//   O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i, m = max_i m_i, over the parts of a unit in order.
// Few rows: block (x, y) has the units that are cut at the ends of shares x, x + gridDim.x, ...; a lane has four channels (two times four
// beyond 128) of a row, eight parts' loads are in flight at a time.  With `many` parts a block works on one row, every warp on every
// eighth part; otherwise a warp on one row.
constexpr int kJoinThreads = 256;
template <typename T, int QUADS>
__global__ void __launch_bounds__(kJoinThreads, QUADS == 1 ? 4 : 2) join_few_kernel(const __grid_constant__ CachedP p, int many, int shares) {
  __shared__ float4 sums[8][32 * QUADS];
  __shared__ float2 stat[8];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quads = p.D / 4;
  const int mine = (int)blockIdx.x + lane * (int)gridDim.x;  // gridDim.x >= shares / 32
  unsigned cut_here = __ballot_sync(0xffffffffu, mine < shares && p.seams[mine].parts > 1);
  for (; cut_here != 0; cut_here &= cut_here - 1) {
    const int share = (int)blockIdx.x + (__ffs(cut_here) - 1) * (int)gridDim.x;
    const Seam j = p.seams[share];
    const int r = many ? (int)blockIdx.y : (int)blockIdx.y * 8 + warp, row = j.r0 + r;
    if (many != 0 && row >= p.N * p.G) continue;
    const bool exists = r < p.rows && row < p.N * p.G, ok = exists && r < j.rows;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o[QUADS];
#pragma unroll
    for (int v = 0; v < QUADS; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int step = many ? 8 : 1;
    for (int k0 = many ? warp : 0; k0 < j.parts && ok; k0 += 8 * step) {
      float2 ml[8];
      float4 x[8][QUADS];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int k = k0 + step * u;
        ml[u] = make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int v = 0; v < QUADS; ++v) x[u][v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < j.parts) {
          const long long at = (long long)(k == 0 ? j.slot0 : 2 * (share + k)) * p.rows + r;
          ml[u] = p.part_ml[at];
#pragma unroll
          for (int v = 0; v < QUADS; ++v)
            if (lane + 32 * v < quads) x[u][v] = *reinterpret_cast<const float4*>(p.part_o + at * p.D + (lane + 32 * v) * 4);
        }
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, ml[u].x);
      const float safe = top == -CUDART_INF_F ? 0.f : top;  // nothing was seen, or nothing but NaN: the sums know
      const float a = exp2f(m - safe);
      m = top;
      l *= a;
#pragma unroll
      for (int v = 0; v < QUADS; ++v) o[v].x *= a, o[v].y *= a, o[v].z *= a, o[v].w *= a;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = exp2f(ml[u].x - safe);
        l = fmaf(w, ml[u].y, l);
#pragma unroll
        for (int v = 0; v < QUADS; ++v) {
          o[v].x = fmaf(w, x[u][v].x, o[v].x); o[v].y = fmaf(w, x[u][v].y, o[v].y);
          o[v].z = fmaf(w, x[u][v].z, o[v].z); o[v].w = fmaf(w, x[u][v].w, o[v].w);
        }
      }
    }
    if (many) {  // the warps' sums become the first warp's
      __syncthreads();  // those of the unit before have been read
#pragma unroll
      for (int v = 0; v < QUADS; ++v) sums[warp][lane + 32 * v] = o[v], o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane == 0) stat[warp] = make_float2(m, l);
      __syncthreads();
      if (warp != 0) continue;
      m = -CUDART_INF_F;
      l = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) m = fmaxf(m, stat[w].x);
      const float safe = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float a = exp2f(stat[w].x - safe);
        l = fmaf(a, stat[w].y, l);
#pragma unroll
        for (int v = 0; v < QUADS; ++v) {
          const float4 y = sums[w][lane + 32 * v];
          o[v].x = fmaf(a, y.x, o[v].x); o[v].y = fmaf(a, y.y, o[v].y); o[v].z = fmaf(a, y.z, o[v].z); o[v].w = fmaf(a, y.w, o[v].w);
        }
      }
    }
    if (!exists) continue;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int i = row / p.G, h = j.head * p.G + row % p.G;
    T* to = o_row<T>(p, j.b, h, i);
#pragma unroll
    for (int v = 0; v < QUADS; ++v)
      if (lane + 32 * v < quads) store4<T>(p, to, (lane + 32 * v) * 4, o[v].x * inv, o[v].y * inv, o[v].z * inv, o[v].w * inv);
    if (lane == 0) store_lse(p, j.b, h, i, ok, m, l);
  }
}

// Many rows: lanes over 32 rows (as the parts lie), a warp for eight channels at a time.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_many_kernel(const __grid_constant__ CachedP p) {
  pdl_wait();
  const Seam j = p.seams[blockIdx.x];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = (int)blockIdx.y * 32 + lane, row = j.r0 + r;
  if (j.parts < 2 || r >= p.rows || row >= p.N * p.G) return;
  const int i = row / p.G, h = j.head * p.G + row % p.G;
  const bool ok = r < j.rows;
  auto slot = [&](int k) -> long long { return k == 0 ? j.slot0 : 2 * ((int)blockIdx.x + k); };
  float m = -CUDART_INF_F, l = 0.f;
#pragma unroll 4
  for (int k = 0; k < (ok ? j.parts : 0); ++k) {
    const float2 x = p.part_ml[slot(k) * p.rows + r];
    const float top = fmaxf(m, x.x), safe = top == -CUDART_INF_F ? 0.f : top;
    l = l * exp2f(m - safe) + exp2f(x.x - safe) * x.y;
    m = top;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T* to = o_row<T>(p, j.b, h, i);
  for (int d = warp * 8; d < p.D; d += 64) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
    for (int k = 0; k < (m != -CUDART_INF_F ? j.parts : 0); ++k) {
      const float w = exp2f(p.part_ml[slot(k) * p.rows + r].x - m);
      const float4* x = reinterpret_cast<const float4*>(p.part_o) + (slot(k) * (p.D / 4) + d / 4) * p.rows + r;
      const float4 y = x[0], z = x[p.rows];
      a.x = fmaf(w, y.x, a.x); a.y = fmaf(w, y.y, a.y); a.z = fmaf(w, y.z, a.z); a.w = fmaf(w, y.w, a.w);
      b.x = fmaf(w, z.x, b.x); b.y = fmaf(w, z.y, b.y); b.z = fmaf(w, z.z, b.z); b.w = fmaf(w, z.w, b.w);
    }
    store4<T>(p, to, d, a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    store4<T>(p, to, d + 4, b.x * inv, b.y * inv, b.z * inv, b.w * inv);
  }
  if (warp == 0) store_lse(p, j.b, h, i, ok, m, l);
}

}  // namespace cache
}  // namespace chill
