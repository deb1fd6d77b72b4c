// Pages that several requests hold (chill_pages_fork, chill_pages_trim_shared), pages that move together (chill_pages_compact), and the copies that both
// ask for (chill_cache_copy).  include/chill_decode.h says what they do.
#include <cooperative_groups.h>

#include "decode_common.cuh"

namespace chill {
namespace decode {
namespace cg = cooperative_groups;

constexpr int kPageThreads = 1024;
constexpr int kPageWarps = kPageThreads / 32;
constexpr int kPageCtas = 8;
constexpr int kMaxCtas = 16;
constexpr int kForkRequests = 8192;
constexpr int kMostPages = 1 << 30;  // the number of a page and what a cluster's CTAs step beyond it fit 32 bits
constexpr int kMostShared = 200 * 1024;
constexpr size_t kUnasked = 40 * 1024;  // dynamic shared memory that every kernel here gets beside its static one

struct ShareP {
  int B, page, num_pages, width;
  int* table;
  long long table_sb;
  int *held, *free_pages, *n_free, *shared;
  const int* lens;
  int* missing;
  const int* parents;
  int* out_lens;
  int *source, *target, *rows, *count;
  int orders;
  int *before, *bits, *state;  // workspace: the tables as they were and a bit for every entry, where they are too large for shared memory; fork: [B][2] what rows held; compact:
                               // [num_pages] where a page goes
};

// Exclusive prefix sum of one value per thread; `total` is the block's sum.
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int sums[kPageWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the sums of the call before this one have been read
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  const int s = lane < (int)(blockDim.x >> 5) ? sums[lane] : 0;
  int y = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  total = __shfl_sync(0xffffffffu, y, 31);
  return __shfl_sync(0xffffffffu, y - s, warp) + x - v;
}

// ------------------------------------------------------------------------------------------------------------ fork / trim
// A row r of the old tables with L tokens in h blocks: `whole` = L / page blocks are full, `rest` = L % page rows of the next one are written.  With c_r
// children, its whole pages get c_r - 1 holders more.  Its begun page stays with the first child where shared = 0, else row r lets go of
// it.  What it lets go of is always a run of blocks [begin, h): all of them without children, else those from `whole` or from the block behind the
// begun one on.  (trim: every row is its own only child, and keeps its begun page.)
//
// Which of the rows that let go of a page puts it on the stack must not depend on the order of the atomics: the counts are worked out first; below zero means
// that nobody holds the page, and then every row that let go of it writes the number of its entry, the first (lowest) one stays.  The word of
// shared[] takes both: -1 for a page without holders, -2 - (entries - 1 - entry) for the claims, of which the minimum is the lowest entry.
//
// Latency is all there is: one cluster, whose barriers separate the steps, and few trips to memory one after the other.  Every CTA has a share of the rows and keeps them as they
// were in shared memory, where children in other CTAs find them too (in the workspace where they are too large: kInside false); what goes back is noted there in bits.
// 4 beams of 700 tokens in pages of 16: 11 us (two of them a launch); 16 groups of 16 beams of up to 16384 tokens (256 rows of 1026 blocks): 29 us in a cluster of 16 CTAs (8: 38), of which the rows' way into
// shared memory 5, counts 3, claims 6 (scattered reads of shared), new tables 4, barriers 4.  Row by row with an atomic for every entry, and the rows in the workspace: 53 us.

// A cluster's barrier costs one CTA alone 0.5 us more than its own.
__device__ __forceinline__ void sync_all(const cg::cluster_group& cluster, int ctas) {
  if (ctas > 1) cluster.sync();
  else __syncthreads();
}

// Rows that a warp has at a time, 32 blocks of each: what neighbouring rows share (the beams of a request, nearly everything) is counted in registers before it is
// counted in memory.
constexpr int kRows = 8;

template <bool kTrim, bool kInside>
__global__ void __launch_bounds__(kPageThreads) share_kernel(const __grid_constant__ ShareP p) {
  extern __shared__ int dynamic[];
  __shared__ int own_total;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = (int)blockDim.x, warps = threads >> 5;
  const int per = ((p.B + ctas - 1) / ctas + kRows - 1) / kRows * kRows, r0 = imin(cta * per, p.B), r1 = imin(r0 + per, p.B);
  const int words = (p.width + 31) / 32;  // of 32 blocks
  // Of this CTA's rows as they were: blocks they hold, those of the run that they let go of begin where, how many go back to the stack (later: before them)
  int *const held = dynamic, *const begin = held + per, *const number = begin + per;
  // fork: blocks that a row's children share; of a row as it will be: the parent (-1: none), its whole blocks, all blocks, the page of the last one
  int *const whole = number + per, *const parent = whole + per, *const taken_over = parent + per, *const now = taken_over + per, *const begun = now + per;
  int *const children = begun + per, *const first = children + p.B;  // fork, [B]: of every row, how many and the first
  int* const rows_inside = kTrim ? whole : first + p.B;              // [per][width]
  int* const back = kInside ? rows_inside + (size_t)per * p.width : p.bits + (size_t)r0 * words;  // [per][words]: bits of the blocks whose pages go back
  const long long entries = (long long)p.B * p.width;
  int2* const summary = reinterpret_cast<int2*>(p.state);
  const int n_free = imin(imax(*p.n_free, 0), p.num_pages);
  auto is_page = [&](int q) { return q >= 0 && q < p.num_pages; };
  auto before = [&](int r) -> int* {  // of this CTA's rows
    return kInside ? rows_inside + (size_t)(r - r0) * p.width : (kTrim ? p.table + r * p.table_sb : p.before + (long long)r * p.width);
  };
  // A warp has a block of kRows rows and some of their words of 32 blocks, every `stride`-th from `word` on
  const int row_blocks = (r1 - r0 + kRows - 1) / kRows, stride = row_blocks > 0 ? imax(warps / row_blocks, 1) : 1;
  auto sweep = [&](auto body) {
    for (int unit = warp; unit < row_blocks * stride; unit += warps) body(r0 + unit % row_blocks * kRows, unit / row_blocks);
  };

  // The rows as they are
  if constexpr (!kTrim || kInside) {
    sweep([&](int rows, int word) {
      for (int j = word * 32 + lane; j < p.width; j += stride * 32) {
        int q[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) q[u] = rows + u < r1 ? p.table[(rows + u) * p.table_sb + j] : -1;
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (rows + u < r1) before(rows + u)[j] = q[u];
      }
    });
  }
  if constexpr (!kTrim) {
    for (int r = threadIdx.x; r < p.B; r += threads) {
      children[r] = 0;
      first[r] = p.B;
    }
  }
  for (int r = r0 + threadIdx.x; r < r1; r += threads) {
    const int i = r - r0, len = clamp_len(p.lens[r]);
    held[i] = imin(imax(p.held[r], 0), p.width);
    if constexpr (kTrim) {
      begin[i] = imin((len + p.page - 1) / p.page, held[i]);
    } else {
      begin[i] = imin(len, held[i] * p.page);  // for now: its tokens
    }
    number[i] = 0;
  }
  __syncthreads();
  if constexpr (!kTrim) {
    for (int b = threadIdx.x; b < p.B; b += threads) {
      const int r = p.parents[b];
      if (r < 0 || r >= p.B) continue;
      atomicAdd(&children[r], 1);
      atomicMin(&first[r], b);
    }
    // What children need to know of a row, in two words: its tokens, and its begun page: stays with the first child (page), goes (-2 - page), none (-1).  Tokens of
    // a begun block without a page are not there.
    for (int r = r0 + threadIdx.x; r < r1; r += threads) {
      const int i = r - r0, len = begin[i], full = len / p.page;
      int2 s = make_int2(full * p.page, -1);
      if (len != s.x) {
        const int q = before(r)[full];
        if (is_page(q)) s = make_int2(len, p.shared[q] == 0 ? q : -2 - q);
      }
      summary[r] = s;
    }
    sync_all(cluster, ctas);  // what rows held is written down
    for (int r = r0 + threadIdx.x; r < r1; r += threads) {
      const int i = r - r0;
      const int2 s = summary[r];
      whole[i] = children[r] > 0 ? s.x / p.page : 0;
      begin[i] = children[r] > 0 && s.x % p.page != 0 && s.y >= 0 ? whole[i] + 1 : whole[i];
    }
    __syncthreads();
  }

  // Counts of holders
  sweep([&](int rows, int word) {
    // of the rows: children beyond one and for how many blocks they count, the run
    int more[kRows], until[kRows], lo[kRows], hi[kRows], top = 0;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int i = rows + u - r0;
      const bool is_row = rows + u < r1;
      more[u] = !kTrim && is_row ? children[rows + u] - 1 : 0;
      until[u] = more[u] > 0 ? whole[i] : 0;
      lo[u] = is_row ? begin[i] : 0;
      hi[u] = is_row ? held[i] : 0;
      top = imax(top, imax(until[u], lo[u] < hi[u] ? hi[u] : 0));
    }
    for (int j = word * 32 + lane; j < top; j += stride * 32) {
      int page = -1, sum = 0;
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const bool goes = j >= lo[u] && j < hi[u];
        if (j >= until[u] && !goes) continue;
        const int q = before(rows + u)[j];
        if (!is_page(q)) continue;
        if (q != page) {
          if (sum != 0) atomicAdd(&p.shared[page], sum);
          page = q;
          sum = 0;
        }
        sum += goes ? -1 : more[u];
      }
      if (sum != 0) atomicAdd(&p.shared[page], sum);
    }
  });
  // New pages: for every child but the first, or for all where the page is somebody else's too; requests in order
  int taken = 0;
  if constexpr (!kTrim) {
    for (int base = 0; base < p.B; base += threads) {
      const int b = base + (int)threadIdx.x;
      int r = b < p.B ? p.parents[b] : -1, rest = 0, total;
      if (r >= p.B) r = -1;
      int2 s = make_int2(0, -1);
      if (r >= 0) {
        s = summary[r];
        rest = s.x % p.page;
      }
      const bool asks = rest != 0 && !(s.y >= 0 && first[r] == b);
      const int off = taken + block_scan(asks ? 1 : 0, total);  // pages that the rows before b want
      taken += total;
      if (b < r0 || b >= r1) continue;
      // row b as it will be
      const bool gets = asks && off < n_free, here = rest != 0 && (!asks || gets);
      const int blocks = s.x / p.page, page = gets ? p.free_pages[n_free - 1 - off] : s.y;
      parent[b - r0] = r;
      taken_over[b - r0] = blocks;
      now[b - r0] = blocks + (here ? 1 : 0);
      begun[b - r0] = page;
      p.out_lens[b] = here ? s.x : blocks * p.page;
      if (gets) {
        p.source[off] = s.y >= 0 ? s.y : -2 - s.y;
        p.target[off] = page;
        p.rows[off] = rest;
      }
    }
  }
  sync_all(cluster, ctas);  // the counts are complete

  // Claims to the pages that nobody holds.  `back` notes for whose
  auto claim_of = [&](int r, int j) { return (int)(-1 - entries + ((long long)r * p.width + j)); };
  sweep([&](int rows, int first_word) {
    int lo[kRows], hi[kRows], bottom = p.width, top = 0;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int i = rows + u - r0;
      lo[u] = rows + u < r1 ? begin[i] : 0;
      hi[u] = rows + u < r1 ? held[i] : 0;
      if (lo[u] >= hi[u]) continue;
      bottom = imin(bottom, lo[u]);
      top = imax(top, hi[u]);
    }
    for (int word = first_word; word < words; word += stride) {
      const int j = word * 32 + lane;
      const bool any = word * 32 < top && word * 32 + 32 > bottom;
      int q[kRows], left[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) q[u] = any && j >= lo[u] && j < hi[u] ? before(rows + u)[j] : -1;
#pragma unroll
      for (int u = 0; u < kRows; ++u) left[u] = is_page(q[u]) && (u == 0 || q[u] != q[u - 1]) ? __ldcg(&p.shared[q[u]]) : 0;  // of equal ones the first is the lowest
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (left[u] < 0) atomicMin(&p.shared[q[u]], claim_of(rows + u, j));
        const unsigned who = any ? __ballot_sync(0xffffffffu, left[u] < 0) : 0;
        if (lane == 0 && rows + u < r1) back[(size_t)(rows + u - r0) * words + word] = (int)who;
      }
    }
  });
  // The new tables
  if constexpr (!kTrim) {
    const int got = imin(taken, n_free);
    sweep([&](int rows, int word) {
      const int* from[kRows];  // the parent's row, nullptr: its blocks stay as they are
      int until[kRows], end[kRows], hi[kRows], last[kRows], top = 0;
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int i = rows + u - r0;
        const bool is_row = rows + u < r1;
        const int r = is_row ? parent[i] : -1, owner = r >= 0 ? r / per : 0;
        from[u] = nullptr;
        if (r >= 0 && r != rows + u)
          from[u] = kInside ? cluster.map_shared_rank(rows_inside, owner) + (size_t)(r - owner * per) * p.width : p.before + (long long)r * p.width;
        until[u] = is_row ? taken_over[i] : 0;
        end[u] = is_row ? now[i] : 0;
        hi[u] = is_row ? held[i] : 0;
        last[u] = is_row ? begun[i] : 0;
        top = imax(top, imax(end[u], hi[u]));
      }
      for (int j = word * 32 + lane; j < top; j += stride * 32) {
        int q[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          q[u] = -2;  // stays as it is
          if (j < until[u]) q[u] = from[u] != nullptr ? from[u][j] : -2;
          else if (j < end[u]) q[u] = last[u];
          else if (j < hi[u]) q[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u)
          if (q[u] != -2) p.table[(rows + u) * p.table_sb + j] = q[u];
      }
    });
    for (int i = got + cta * threads + (int)threadIdx.x; i < p.B; i += ctas * threads) {
      p.source[i] = p.target[i] = -1;
      p.rows[i] = 0;
    }
    if (cta == 0 && threadIdx.x == 0) {
      *p.count = got;
      *p.missing = imax(taken - n_free, 0);
    }
  }
  sync_all(cluster, ctas);  // the lowest claims are there; what was taken from the stack, and other CTAs' rows, have been read

  // How many pages every row puts on the stack: those of which its claim is the lowest
  for (int item = warp; item < (r1 - r0) * words; item += warps) {
    const unsigned claims = (unsigned)back[item];
    if (claims == 0) continue;
    const int i = item / words, j = item % words * 32 + lane;
    const bool mine = (claims >> lane & 1) && __ldcg(&p.shared[before(r0 + i)[j]]) == claim_of(r0 + i, j);
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) {
      back[item] = (int)who;
      if (who != 0) atomicAdd(&number[i], __popc(who));
    }
  }
  __syncthreads();
  int own = 0;
  for (int base = 0; base < r1 - r0; base += threads) {
    const int i = base + (int)threadIdx.x;
    int total;
    const int n = i < r1 - r0 ? number[i] : 0, x = block_scan(n, total);
    if (i < r1 - r0) number[i] = n == 0 ? -1 : own + x;  // pages of this CTA's rows before it; -1: it has none itself
    own += total;
  }
  if (threadIdx.x == 0) own_total = own;
  sync_all(cluster, ctas);
  int earlier = 0, all = 0;
  for (int c = 0; c < ctas; ++c) {
    const int n = *cluster.map_shared_rank(&own_total, c);
    if (c < cta) earlier += n;
    all += n;
  }
  const int left = n_free - imin(taken, n_free);
  for (int r = r0 + warp; r < r1; r += warps) {
    const int i = r - r0;
    for (int w0 = 0, at = number[i]; number[i] >= 0 && w0 < words; w0 += 32) {
      unsigned who = w0 + lane < words ? (unsigned)back[(size_t)i * words + w0 + lane] : 0;
      int n = __popc(who), x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      for (int rank = at + x - n; who != 0; who &= who - 1, ++rank) {
        const int q = before(r)[(w0 + lane) * 32 + __ffs(who) - 1];
        const long long to = (long long)left + all - 1 - (earlier + rank);
        if (to >= 0 && to < p.num_pages) p.free_pages[to] = q;  // `held` can be nonsense
        p.shared[q] = 0;
      }
      at += __shfl_sync(0xffffffffu, x, 31);
    }
    if (kTrim) {
      __syncwarp();
      for (int j = begin[i] + lane; j < held[i]; j += 32) p.table[r * p.table_sb + j] = -1;
    }
  }
  for (int b = r0 + threadIdx.x; b < r1; b += threads) p.held[b] = kTrim ? begin[b - r0] : now[b - r0];
  if (cta == 0 && threadIdx.x == 0) *p.n_free = imin(all, p.num_pages - left) + left;
  if (ctas > 1) cluster.sync();  // own_total has been read
}

// ------------------------------------------------------------------------------------------------------------ compact
// With U pages in use, hole i (from below) is the i-th free page below U, and takes what used page i (from above) of those at U and beyond
// holds: as many of both.  One prefix sum over the pages; every CTA of a cluster has a run of them.  6600 pages, 96 rows of 126 blocks: 11 us, six steps with a barrier between.
__global__ void __launch_bounds__(kPageThreads) compact_kernel(const __grid_constant__ ShareP p) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int per = ((p.num_pages + ctas - 1) / ctas + 3) / 4 * 4, p0 = imin(cta * per, p.num_pages), p1 = imin(p0 + per, p.num_pages);
  const int thread = cta * kPageThreads + (int)threadIdx.x, threads = ctas * kPageThreads;
  int* const to = p.state;                      // [num_pages]: -1 free, later where a page goes
  int* const totals = p.state + p.num_pages;    // [ctas]: free pages
  int* const moves = totals + kPageCtas;        // [1]
  const int n_free = imin(imax(*p.n_free, 0), p.num_pages);
  for (int q = p0 + threadIdx.x; q < p1; q += kPageThreads) to[q] = q;
  sync_all(cluster, ctas);
  for (int i = thread; i < n_free; i += threads) {
    const int q = p.free_pages[i];
    if (q >= 0 && q < p.num_pages) to[q] = -1;
  }
  sync_all(cluster, ctas);
  int own = 0;
  for (int q = p0 + threadIdx.x; q < p1; q += kPageThreads) own += __ldcg(&to[q]) < 0 ? 1 : 0;
  int free_here;
  block_scan(own, free_here);
  if (threadIdx.x == 0) totals[cta] = free_here;
  sync_all(cluster, ctas);
  int before = 0, all = 0;
  for (int c = 0; c < ctas; ++c) {
    const int n = __ldcg(&totals[c]);
    if (c < cta) before += n;
    all += n;
  }
  const int used = p.num_pages - all;
  for (int base = p0; base < p1; base += kPageThreads) {
    const int q = base + (int)threadIdx.x;
    const int is_free = q < p1 && __ldcg(&to[q]) < 0 ? 1 : 0;
    int total;
    const int free_before = before + block_scan(is_free, total);
    before += total;
    if (q >= p1) continue;
    if (q < used) {
      if (is_free) p.target[free_before] = q;
    } else if (!is_free) {
      const int above = p.num_pages - 1 - q - (all - free_before);  // used pages above this one
      p.source[above] = q;
      p.rows[above] = p.page;
    }
    if (q == used) *moves = free_before;  // holes
  }
  if (used == p.num_pages && thread == 0) *moves = 0;
  sync_all(cluster, ctas);
  const int count = __ldcg(moves);
  for (int i = thread; i < p.orders; i += threads) {
    if (i < count) {
      const int from = __ldcg(&p.source[i]), at = __ldcg(&p.target[i]);
      to[from] = at;
      if (p.shared != nullptr) {
        p.shared[at] = p.shared[from];
        p.shared[from] = 0;
      }
    } else {
      p.source[i] = p.target[i] = -1;
      p.rows[i] = 0;
    }
  }
  for (int i = thread; i < all; i += threads) p.free_pages[i] = p.num_pages - 1 - i;
  if (thread == 0) {
    *p.count = count;
    *p.n_free = all;
  }
  sync_all(cluster, ctas);
  constexpr int kUnroll = 8;
  const int warp = thread >> 5, warps = threads >> 5, lane = threadIdx.x & 31, pieces = (p.width + 32 * kUnroll - 1) / (32 * kUnroll);
  for (long long item = warp; item < (long long)p.B * pieces; item += warps) {
    const int b = (int)(item / pieces), j0 = (int)(item % pieces) * 32 * kUnroll + lane, held = imin(imax(p.held[b], 0), p.width);
    int* row = p.table + b * p.table_sb;
    int q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = j0 + 32 * u < held ? row[j0 + 32 * u] : -1;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (q[u] < used || q[u] >= p.num_pages) continue;
      const int now = __ldcg(&to[q[u]]);
      if (now >= 0) row[j0 + 32 * u] = now;
    }
  }
}

static size_t workspace_of(const chill_share_args& a) {
  const size_t ints = (size_t)a.B * a.table_width + (size_t)a.B * ((a.table_width + 31) / 32) + 2 * (size_t)a.B + (size_t)a.num_pages + 64;
  return (ints * 4 + 255) / 256 * 256;
}

static int check_share(const chill_share_args* a, bool pointers) {
  if (a == nullptr || a->B <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->table_width <= 0) return CHILL_E_INVALID;
  if (a->B > kMaxRequests || a->num_pages > kMostPages || (long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->table_width * a->page_size > kMaxLen ||
      (long long)a->B * a->table_width > 0x7ffffff0ll)  // the number of an entry is a claim, below -1
    return CHILL_E_TOO_LARGE;
  if (!pointers) return CHILL_OK;
  if (!a->table || !a->held || !a->free_pages || !a->n_free || (a->table_stride < a->table_width && a->B > 1)) return CHILL_E_INVALID;
  if (a->workspace == nullptr || a->workspace_bytes < workspace_of(*a) || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return CHILL_E_INVALID;
  return CHILL_OK;
}

static ShareP share_params(const chill_share_args& a) {
  ShareP p{};
  p.B = a.B; p.page = a.page_size; p.num_pages = a.num_pages; p.width = a.table_width;
  p.table = a.table; p.table_sb = a.table_stride;
  p.held = a.held; p.free_pages = a.free_pages; p.n_free = a.n_free; p.shared = a.shared;
  p.lens = a.lens; p.missing = a.missing; p.parents = a.parents; p.out_lens = a.out_lens;
  p.source = a.source; p.target = a.target; p.rows = a.rows; p.count = a.count;
  p.state = (int*)a.workspace;
  p.before = p.state + 2 * (size_t)a.B;  // fork and trim; compact has the whole of it
  p.bits = p.before + (size_t)a.B * a.table_width;
  return p;
}

template <class F>
static int launch_cluster(F kernel, const ShareP& p, int ctas, int threads, size_t smem, cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  // 48 KB without asking, of which a kernel's static shared memory takes its part.  Always to the same limit: host threads may be here at once
  if (smem > kUnasked) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared);
    if (e != cudaSuccess) return record_cuda_failure(e, what);
  }
  if (ctas > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return record_cuda_failure(e, what);
  }
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return record_cuda_failure(e, what);
  count_launches(1);
  return CHILL_OK;
}

// What a call has to look at: words of 32 blocks of kRows rows.  One CTA of 256 threads for little of it, a cluster of 8 or 16 for more.
struct Shape {
  int ctas, threads;
};
static Shape shape_for(const ShareP& p) {
  const long long items = (long long)((p.B + kRows - 1) / kRows) * ((p.width + 31) / 32);
  if (items <= 16) return {1, 256};
  return {items <= 256 ? kPageCtas : kMaxCtas, kPageThreads};
}

template <bool kTrim>
static int launch_share(const ShareP& p, cudaStream_t st) {
  const Shape s = shape_for(p);
  const int per = ((p.B + s.ctas - 1) / s.ctas + kRows - 1) / kRows * kRows;
  const size_t bytes = (kTrim ? 3 * (size_t)per : 8 * (size_t)per + 2 * (size_t)p.B) * 4, rows = (size_t)per * (p.width + (p.width + 31) / 32) * 4;
  const char* what = kTrim ? "trim launch" : "fork launch";
  if (bytes + rows <= (size_t)kMostShared) return launch_cluster(share_kernel<kTrim, true>, p, s.ctas, s.threads, bytes + rows, st, what);
  return launch_cluster(share_kernel<kTrim, false>, p, s.ctas, s.threads, bytes, st, what);
}

// ------------------------------------------------------------------------------------------------------------ copy
// Orders times layers times kv heads times rows: a copy, bound by memory.  How many orders there are is known on the GPU only, so the grid is as large as the
// GPU and goes over the vectors; nobody looks at orders behind *count.  3060 pages of 32 rows, 8 heads of 128 in bf16, K and V (802 MB read and written): 140 us, 0.88 of a copy's rate;
// a block for each head's part of a page, half of its threads idle there: 173 us.
struct CopyP {
  int layers, Hkv, page, num_pages, orders, per_row;
  char *k, *v;
  long long ks[5], vs[5];  // bytes, the last one of a vector
  const int *source, *target, *rows, *count;
  bool both;
};

constexpr int kCopyThreads = 256, kCopyEach = 4;

template <class V>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyP p) {
  constexpr int kChunk = kCopyThreads * kCopyEach;  // vectors that a block moves at a time, of one page, layer and tensor
  const int count = imin(imax(*p.count, 0), p.orders);
  const long long chunks = ((long long)p.Hkv * p.page * p.per_row + kChunk - 1) / kChunk, items = (long long)count * p.layers * chunks * (p.both ? 2 : 1);
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long at = item / chunks;
    const int chunk = (int)(item - at * chunks), order = (int)(at / p.layers % count), layer = (int)(at % p.layers);
    const bool is_v = at >= (long long)count * p.layers;
    const int from = p.source[order], to = p.target[order], rows = imin(imax(p.rows[order], 0), p.page);
    if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages || from == to) continue;
    const long long* st = is_v ? p.vs : p.ks;
    char* base = (is_v ? p.v : p.k) + layer * st[0];
    const char* src = base + from * st[1];
    char* dst = base + to * st[1];
    const unsigned per_head = (unsigned)rows * (unsigned)p.per_row;
    const unsigned end = (unsigned)p.Hkv * per_head;
    V x[kCopyEach];
    long long offset[kCopyEach];
#pragma unroll
    for (int u = 0; u < kCopyEach; ++u) {
      const unsigned i = (unsigned)chunk * kChunk + u * kCopyThreads + threadIdx.x;
      offset[u] = -1;
      if (i >= end) continue;
      const unsigned h = i / per_head, in_head = i - h * per_head, row = in_head / (unsigned)p.per_row, c = in_head - row * (unsigned)p.per_row;
      offset[u] = h * st[2] + row * st[3] + c * st[4];
      x[u] = load_once<V>(src + offset[u]);
    }
#pragma unroll
    for (int u = 0; u < kCopyEach; ++u)
      if (offset[u] >= 0) store_once(dst + offset[u], x[u]);
  }
}

}  // namespace decode
}  // namespace chill

using namespace chill::decode;

extern "C" {

size_t chill_share_workspace_bytes(const chill_share_args* a) { return check_share(a, false) == CHILL_OK ? workspace_of(*a) : 0; }

int chill_pages_fork(const chill_share_args* a, void* stream) {
  const int st = check_share(a, true);
  if (st != CHILL_OK) return st;
  if (!a->shared || !a->lens || !a->missing || !a->parents || !a->out_lens || !a->source || !a->target || !a->rows || !a->count) return CHILL_E_INVALID;
  if (a->B > kForkRequests) return CHILL_E_TOO_LARGE;
  if (a->out_lens == a->lens || a->out_lens == a->parents) return CHILL_E_INVALID;  // other CTAs read these
  return launch_share<false>(share_params(*a), (cudaStream_t)stream);
}

int chill_pages_trim_shared(const chill_share_args* a, void* stream) {
  const int st = check_share(a, true);
  if (st != CHILL_OK) return st;
  if (!a->shared || !a->lens) return CHILL_E_INVALID;
  return launch_share<true>(share_params(*a), (cudaStream_t)stream);
}

int chill_pages_compact(const chill_share_args* a, void* stream) {
  const int st = check_share(a, true);
  if (st != CHILL_OK) return st;
  if (!a->source || !a->target || !a->rows || !a->count) return CHILL_E_INVALID;
  ShareP p = share_params(*a);
  p.orders = imax(a->num_pages / 2, 1);
  return launch_cluster(compact_kernel, p, a->num_pages <= 2 * kPageThreads && shape_for(p).ctas == 1 ? 1 : kPageCtas, kPageThreads, 0, (cudaStream_t)stream, "compact launch");
}

int chill_cache_copy(const chill_copy_args* a, void* stream) {
  if (a == nullptr || a->layers <= 0 || a->num_pages <= 0 || a->H_kv <= 0 || a->page_size <= 0 || a->D <= 0 || a->orders <= 0) return CHILL_E_INVALID;
  if (!known_dtype(a->dtype)) return CHILL_E_UNSUPPORTED;
  if ((long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->page_size * a->D > (1 << 30) ||
      (long long)a->page_size * a->D * a->H_kv > (1 << 30))
    return CHILL_E_TOO_LARGE;
  if (!a->k_cache || !a->v_cache || !a->source || !a->target || !a->rows || !a->count) return CHILL_E_INVALID;
  const int es = elem_size(a->dtype);
  CopyP p{};
  p.layers = a->layers; p.Hkv = a->H_kv; p.page = a->page_size; p.num_pages = a->num_pages; p.orders = a->orders;
  p.k = (char*)a->k_cache; p.v = (char*)a->v_cache;
  p.source = a->source; p.target = a->target; p.rows = a->rows; p.count = a->count;
  p.both = a->k_cache != a->v_cache;
  for (int d = 0; d < 5 && !p.both; ++d)  // one tensor for both: each row moves once
    if (a->k_cache_strides[d] != a->v_cache_strides[d]) return CHILL_E_INVALID;
  int vec = imin(row_vector(a->k_cache, a->k_cache_strides, 4, es), row_vector(a->v_cache, a->v_cache_strides, 4, es));
  while (vec > es && a->D * es % vec != 0) vec /= 2;
  if (vec < 16) vec = es;
  p.per_row = a->D * es / vec;
  for (int d = 0; d < 5; ++d) {
    p.ks[d] = (long long)a->k_cache_strides[d] * es;
    p.vs[d] = (long long)a->v_cache_strides[d] * es;
  }
  if (vec == 16) p.ks[4] = p.vs[4] = 16;
  const dim3 grid((unsigned)(8 * sm_count()));
  if (vec == 16) copy_kernel<uint4><<<grid, kCopyThreads, 0, (cudaStream_t)stream>>>(p);
  else if (es == 4) copy_kernel<uint32_t><<<grid, kCopyThreads, 0, (cudaStream_t)stream>>>(p);
  else copy_kernel<uint16_t><<<grid, kCopyThreads, 0, (cudaStream_t)stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_cuda_failure(e, "copy launch");
  count_launches(1);
  return CHILL_OK;
}

}  // extern "C"
