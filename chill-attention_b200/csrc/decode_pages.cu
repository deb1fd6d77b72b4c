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
constexpr int kForkRequests = 8192;

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
  int *before, *state;  // workspace: fork: the tables as they were, [B][2] what rows held; compact: [num_pages] where a page goes
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
  const int s = sums[lane];
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
// children, its whole pages get c_r - 1 holders more.  Its begun page stays with the first child where shared = 0 (row_keeps), else row r lets go of
// it.  What it lets go of is always a run of blocks [begin, h): all of them without children, else those from `whole` or from the block behind the
// begun one on.  (trim: every row is its own only child, and keeps its begun page.)
//
// Which of the rows that let go of a page puts it on the stack must not depend on the order of the atomics: the counts are worked out first; below zero means
// that nobody holds the page, and then every row that let go of it writes the number of its entry, the first (lowest) one stays.  The word of
// shared[] takes both: -1 for a page without holders, -2 - (entries - 1 - entry) for the claims, of which the minimum is the lowest entry.
//
// Latency is all there is: one cluster, whose barriers separate the steps.  Every CTA has a share of the rows, a warp goes over a row.
struct Row {
  int held, len, whole, rest, page;  // page: of the begun block, -1 where there is none
};

__device__ __forceinline__ Row row_of(const ShareP& p, int r) {
  Row x;
  x.held = imin(imax(p.held[r], 0), p.width);
  x.len = (int)imin((long long)clamp_len(p.lens[r]) < (long long)x.held * p.page ? clamp_len(p.lens[r]) : x.held * p.page, kMaxLen);
  x.whole = x.len / p.page;
  x.rest = x.len - x.whole * p.page;
  x.page = -1;
  if (x.rest > 0) {
    const int q = p.table[r * p.table_sb + x.whole];
    if (q >= 0 && q < p.num_pages) x.page = q;
  }
  return x;
}

// What children need to know of a row, in two words: its tokens, and its begun page: stays with the first child (page), goes (-2 - page), none (-1).
// Tokens of a begun block without a page are not there.
__device__ __forceinline__ int2 summary_of(const ShareP& p, const Row& x) {
  if (x.page < 0) return make_int2(x.whole * p.page, -1);
  return make_int2(x.len, p.shared[x.page] == 0 ? x.page : -2 - x.page);
}

// Blocks of a row that a lane has at a time: as many loads on their way.
constexpr int kUnroll = 8;

template <bool kTrim>
__global__ void __launch_bounds__(kPageThreads) share_kernel(const __grid_constant__ ShareP p) {
  extern __shared__ int dynamic[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (p.B + ctas - 1) / ctas, r0 = imin(cta * per, p.B), r1 = imin(r0 + per, p.B);
  int* const number = dynamic;                 // [per]: of this CTA's rows, see below
  int* const children = dynamic + per;         // [B], fork
  int* const first = dynamic + per + p.B;      // [B], fork: the first child
  const long long entries = (long long)p.B * p.width;
  int2* const summary = reinterpret_cast<int2*>(p.state);
  int* const totals = p.state + (kTrim ? 0 : 2 * p.B);
  const int n_free = imin(imax(*p.n_free, 0), p.num_pages);
  // Warps go over pieces of rows: 32 * kUnroll blocks
  const int pieces = (p.width + 32 * kUnroll - 1) / (32 * kUnroll);
  auto is_page = [&](int q) { return q >= 0 && q < p.num_pages; };
  auto held_of = [&](int r) { return imin(imax(p.held[r], 0), p.width); };
  auto table_before = [&](int r) { return kTrim ? p.table + r * p.table_sb : p.before + (long long)r * p.width; };

  if constexpr (!kTrim) {
    for (int r = threadIdx.x; r < p.B; r += kPageThreads) {
      children[r] = 0;
      first[r] = p.B;
    }
    for (int r = r0 + threadIdx.x; r < r1; r += kPageThreads) summary[r] = summary_of(p, row_of(p, r));
    for (int item = warp; item < (r1 - r0) * pieces; item += kPageWarps) {
      const int r = r0 + item / pieces, j0 = item % pieces * 32 * kUnroll + lane, held = held_of(r);
      int q[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) q[u] = j0 + 32 * u < held ? p.table[r * p.table_sb + j0 + 32 * u] : -1;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j0 + 32 * u < held) p.before[(long long)r * p.width + j0 + 32 * u] = q[u];
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.B; b += kPageThreads) {
      const int r = p.parents[b];
      if (r < 0 || r >= p.B) continue;
      atomicAdd(&children[r], 1);
      atomicMin(&first[r], b);
    }
    cluster.sync();  // what rows held is written down
  }

  // Row r: `whole` blocks that its children share, the run [begin, held) that it lets go of.
  auto run_of = [&](int r, int& whole, int& begin, int& held) {
    held = held_of(r);
    if constexpr (kTrim) {
      whole = 0;
      begin = imin((clamp_len(p.lens[r]) + p.page - 1) / p.page, held);
    } else {
      const int2 s = summary[r];
      const bool begun = s.x % p.page != 0;
      whole = children[r] > 0 ? s.x / p.page : 0;
      begin = children[r] > 0 ? whole + (begun && s.y >= 0 ? 1 : 0) : 0;
    }
  };

  // Counts of holders
  for (int item = warp; item < (r1 - r0) * pieces; item += kPageWarps) {
    const int r = r0 + item / pieces, j0 = item % pieces * 32 * kUnroll + lane;
    int whole, begin, held;
    run_of(r, whole, begin, held);
    const int more = kTrim ? 0 : children[r] - 1;
    if (more <= 0) whole = 0;
    int q[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int j = j0 + 32 * u;
      q[u] = j < whole || (j >= begin && j < held) ? table_before(r)[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (is_page(q[u])) atomicAdd(&p.shared[q[u]], j0 + 32 * u < whole ? more : -1);
  }
  // New pages: for every child but the first, or for all where the page is somebody else's too; requests in order
  int taken = 0;
  auto parent_of = [&](int b) {
    const int r = p.parents[b];
    return r >= 0 && r < p.B ? r : -1;
  };
  auto wants = [&](int b, int r) {
    if (r < 0) return false;
    const int2 s = summary[r];
    return s.x % p.page != 0 && !(s.y >= 0 && first[r] == b);
  };
  if constexpr (!kTrim) {
    for (int base = 0; base < p.B; base += kPageThreads) {
      const int b = base + (int)threadIdx.x;
      int total;
      const int x = block_scan(b < p.B && wants(b, parent_of(b)) ? 1 : 0, total);
      if (b >= r0 && b < r1) number[b - r0] = taken + x;  // pages that the rows before b want
      taken += total;
    }
  }
  cluster.sync();  // the counts are complete

  // Claims to the pages that nobody holds
  auto claim_of = [&](int r, int j) { return (int)(-1 - entries + ((long long)r * p.width + j)); };
  for (int item = warp; item < (r1 - r0) * pieces; item += kPageWarps) {
    const int r = r0 + item / pieces, j0 = item % pieces * 32 * kUnroll + lane;
    int whole, begin, held;
    run_of(r, whole, begin, held);
    int q[kUnroll], left[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) q[u] = j0 + 32 * u >= begin && j0 + 32 * u < held ? table_before(r)[j0 + 32 * u] : -1;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) left[u] = is_page(q[u]) ? __ldcg(&p.shared[q[u]]) : 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (left[u] < 0) atomicMin(&p.shared[q[u]], claim_of(r, j0 + 32 * u));
  }
  // The new tables
  if constexpr (!kTrim) {
    const int got = imin(taken, n_free);
    for (int item = warp; item < (r1 - r0) * pieces; item += kPageWarps) {
      const int b = r0 + item / pieces, j0 = item % pieces * 32 * kUnroll + lane, held = held_of(b), r = parent_of(b);
      const int2 s = r >= 0 ? summary[r] : make_int2(0, -1);
      const int whole = s.x / p.page, rest = s.x - whole * p.page, off = number[b - r0];
      const bool asks = wants(b, r), here = rest > 0 && (!asks || off < got);
      const int begun = asks && here ? p.free_pages[n_free - 1 - off] : s.y, now = whole + (here ? 1 : 0);
      int* to = p.table + b * p.table_sb;
      int q[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) q[u] = j0 + 32 * u < whole && r != b ? p.before[(long long)r * p.width + j0 + 32 * u] : begun;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int j = j0 + 32 * u;
        if (j < now) {
          if (j >= whole || r != b) to[j] = q[u];
        } else if (j < held) {
          to[j] = -1;
        }
      }
      if (item % pieces == 0 && lane == 0) {
        p.out_lens[b] = here ? s.x : whole * p.page;
        if (asks && here) {
          p.source[off] = -2 - (s.y >= 0 ? -2 - s.y : s.y);
          p.target[off] = begun;
          p.rows[off] = rest;
        }
      }
    }
    for (int i = got + cta * kPageThreads + (int)threadIdx.x; i < p.B; i += ctas * kPageThreads) {
      p.source[i] = p.target[i] = -1;
      p.rows[i] = 0;
    }
    if (cta == 0 && threadIdx.x == 0) {
      *p.count = got;
      *p.missing = imax(taken - n_free, 0);
    }
  }
  cluster.sync();  // the lowest claims are there; what was taken from the stack has been read

  // How many pages every row puts on the stack
  auto goes_back = [&](int r, int j, int q) { return is_page(q) && __ldcg(&p.shared[q]) == claim_of(r, j); };
  for (int r = r0 + warp; r < r1; r += kPageWarps) {
    int whole, begin, held, n = 0;
    run_of(r, whole, begin, held);
    for (int j = begin + lane; j < held; j += 32) n += goes_back(r, j, table_before(r)[j]) ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    __syncwarp();
    if (lane == 0) number[r - r0] = n;
  }
  __syncthreads();
  int own = 0;
  for (int base = 0; base < r1 - r0; base += kPageThreads) {
    const int i = base + (int)threadIdx.x;
    int total;
    const int n = i < r1 - r0 ? number[i] : 0, x = block_scan(n, total);
    if (i < r1 - r0) number[i] = n == 0 ? -1 : own + x;  // pages of this CTA's rows before it, -1: none of its own
    own += total;
  }
  if (threadIdx.x == 0) totals[cta] = own;
  cluster.sync();
  int earlier = 0, all = 0;
  for (int c = 0; c < ctas; ++c) {
    const int n = __ldcg(&totals[c]);
    if (c < cta) earlier += n;
    all += n;
  }
  const int left = n_free - imin(taken, n_free);
  for (int r = r0 + warp; r < r1; r += kPageWarps) {
    int whole, begin, held;
    run_of(r, whole, begin, held);
    int at = number[r - r0];
    if (at < 0 && !kTrim) begin = held;
    at += earlier;
    const int* old = table_before(r);
    for (int j0 = begin; j0 < held; j0 += 32) {
      const int j = j0 + lane, q = j < held ? old[j] : -1;
      const bool back = goes_back(r, j, q);
      const unsigned who = __ballot_sync(0xffffffffu, back);
      if (back) {
        const long long to = (long long)left + all - 1 - (at + __popc(who & ((1u << lane) - 1)));
        if (to >= 0 && to < p.num_pages) p.free_pages[to] = q;  // `held` can be nonsense
        p.shared[q] = 0;
      }
      at += __popc(who);
      if (kTrim && j < held) p.table[r * p.table_sb + j] = -1;
    }
  }
  __syncthreads();  // `held` has been read
  for (int b = r0 + threadIdx.x; b < r1; b += kPageThreads) {
    if constexpr (kTrim) {
      p.held[b] = imin(held_of(b), (clamp_len(p.lens[b]) + p.page - 1) / p.page);
    } else {
      p.held[b] = (p.out_lens[b] + p.page - 1) / p.page;
    }
  }
  if (cta == 0 && threadIdx.x == 0) *p.n_free = imin(all, p.num_pages - left) + left;
}

// ------------------------------------------------------------------------------------------------------------ compact
// With U pages in use, hole i (from below) is the i-th free page below U, and takes what used page i (from above) of those at U and beyond
// holds: as many of both.  One prefix sum over the pages; every CTA of a cluster has a run of them.
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
  cluster.sync();
  for (int i = thread; i < n_free; i += threads) {
    const int q = p.free_pages[i];
    if (q >= 0 && q < p.num_pages) to[q] = -1;
  }
  cluster.sync();
  int own = 0;
  for (int q = p0 + threadIdx.x; q < p1; q += kPageThreads) own += __ldcg(&to[q]) < 0 ? 1 : 0;
  int free_here;
  block_scan(own, free_here);
  if (threadIdx.x == 0) totals[cta] = free_here;
  cluster.sync();
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
  cluster.sync();
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
  cluster.sync();
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
  const size_t ints = (size_t)a.B * a.table_width + 2 * (size_t)a.B + 2 + (size_t)a.num_pages + 64;
  return (ints * 4 + 255) / 256 * 256;
}

static int check_share(const chill_share_args* a, bool pointers) {
  if (a == nullptr || a->B <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->table_width <= 0) return CHILL_E_INVALID;
  if (a->B > kMaxRequests || (long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->table_width * a->page_size > kMaxLen ||
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
  p.before = p.state + 2 * ((size_t)a.B + 1) + 62;
  return p;
}

template <class F>
static int launch_cluster(F kernel, const ShareP& p, int ctas, size_t smem, cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return record_cuda_failure(e, what);
  }
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kPageThreads);
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

// One CTA where a warp has a piece of a row each, a cluster for more.
static int ctas_for(const ShareP& p) {
  const long long pieces = (long long)p.B * ((p.width + 32 * kUnroll - 1) / (32 * kUnroll));
  return pieces <= kPageWarps ? 1 : kPageCtas;
}

template <bool kTrim>
static int launch_share(const ShareP& p, cudaStream_t st) {
  const int ctas = ctas_for(p), per = (p.B + ctas - 1) / ctas;
  return launch_cluster(share_kernel<kTrim>, p, ctas, ((size_t)per + (kTrim ? 0 : 2 * (size_t)p.B)) * 4, st, kTrim ? "trim launch" : "fork launch");
}

// ------------------------------------------------------------------------------------------------------------ copy
// Orders times layers times kv heads times rows: a copy, bound by memory.  How many orders there are is known on the GPU only, so the grid is as large as the
// GPU and goes over the vectors; nobody looks at orders behind *count.
struct CopyP {
  int layers, Hkv, page, num_pages, orders, per_row;
  char *k, *v;
  long long ks[5], vs[5];  // bytes, the last one of a vector
  const int *source, *target, *rows, *count;
  bool both;
};

template <class V>
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ CopyP p) {
  const int count = imin(imax(*p.count, 0), p.orders);
  const long long per_head = (long long)p.page * p.per_row;               // vectors of a kv head's part of a page
  const long long chunks = (per_head + 1023) / 1024;                      // a block moves 1024 of them
  const long long items = (long long)count * p.layers * p.Hkv * chunks * (p.both ? 2 : 1);
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    long long at = item;
    const int chunk = (int)(at % chunks);
    at /= chunks;
    const int h = (int)(at % p.Hkv);
    at /= p.Hkv;
    const int layer = (int)(at % p.layers);
    at /= p.layers;
    const int order = (int)(at % count);
    const bool is_v = at >= count;
    const int from = p.source[order], to = p.target[order], rows = imin(imax(p.rows[order], 0), p.page);
    if (from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages || from == to) continue;
    const long long* st = is_v ? p.vs : p.ks;
    char* base = (is_v ? p.v : p.k) + layer * st[0] + h * st[2];
    const char* src = base + from * st[1];
    char* dst = base + to * st[1];
    const int end = rows * p.per_row;
    V x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = chunk * 1024 + u * 256 + (int)threadIdx.x, row = i / p.per_row, c = i - row * p.per_row;
      if (i < end) x[u] = *reinterpret_cast<const V*>(src + row * st[3] + c * st[4]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = chunk * 1024 + u * 256 + (int)threadIdx.x, row = i / p.per_row, c = i - row * p.per_row;
      if (i < end) *reinterpret_cast<V*>(dst + row * st[3] + c * st[4]) = x[u];
    }
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
  return launch_cluster(compact_kernel, p, a->num_pages <= 2 * kPageThreads && ctas_for(p) == 1 ? 1 : kPageCtas, 0, (cudaStream_t)stream, "compact launch");
}

int chill_cache_copy(const chill_copy_args* a, void* stream) {
  if (a == nullptr || a->layers <= 0 || a->num_pages <= 0 || a->H_kv <= 0 || a->page_size <= 0 || a->D <= 0 || a->orders <= 0) return CHILL_E_INVALID;
  if (!known_dtype(a->dtype)) return CHILL_E_UNSUPPORTED;
  if ((long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->page_size * a->D > (1 << 30)) return CHILL_E_TOO_LARGE;
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
  if (vec == 16) copy_kernel<uint4><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else if (es == 4) copy_kernel<uint32_t><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else copy_kernel<uint16_t><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_cuda_failure(e, "copy launch");
  count_launches(1);
  return CHILL_OK;
}

}  // extern "C"
