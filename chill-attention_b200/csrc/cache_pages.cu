// Pages of a key / value cache, kept on the GPU: which pages a request holds (table), which are free (a stack), where new tokens
// go (slots), their positions and, for a tree of drafted tokens, their ancestors; the kernels that store new rows at their slots
// and that move the accepted path of a tree together.  Entry points: chill_pages_reserve / _trim, chill_cache_append / _commit
// (include/chill_cache.h).  Nothing here depends on the mask.
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "cache_common.cuh"
#include "chill_cache.h"

namespace chill {

int record_cuda_failure(cudaError_t e, const char* what);  // cache_abi.cu
void count_launches(int n);                                // cache_abi.cu

namespace cache {

// ------------------------------------------------------------------------------------------------ reserve / trim
// reserve:  need_b = pages of lens[b] + new[b] tokens, take_b = max(0, need_b - held_b), off_b = sum of take over the requests
//           before b; the j-th page taken for b is free[n_free - 1 - (off_b + j)], while there is one.
// trim:     give_b = max(0, held_b - pages of lens[b]), r_b = sum of give before b, K = all; the j-th page given back by b goes to
//           free[n_free + K - 1 - (r_b + j)]: the exact inverse, so pages that were reserved last come first again.
// Both are one prefix sum over the requests and a few words for each: latency is all there is.  One launch; its first cluster has
// the pages: every CTA sums up the requests before its own ones (they are a few KB in L2), the cluster barrier separates these reads
// of `held` and `n_free` from the writes to them, and after it each CTA works on its own share of the requests.  Further clusters
// work out positions and ancestors, which do not depend on pages, beside it.
constexpr int kPageThreads = 1024;
constexpr int kPageCtas = 8;             // CTAs of the cluster (one where there is little to write)
constexpr int kMaxRequests = 65535;      // check_pages
constexpr int kOwnRequests = (kMaxRequests + kPageCtas - 1) / kPageCtas;

struct PagesP {
  int B, N, page, num_pages, width, words;
  int* table;
  long long table_sb;
  int *held, *free_pages, *n_free, *missing;
  const int *lens, *new_lens, *parents;
  int *slots, *positions, *ancestors;
  int* stored;  // may be null
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive prefix sum of one value per thread; `total` is the block's sum.
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int sums[kPageThreads / 32];
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
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPageThreads / 32; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return before + x - v;
}

// Pages request b holds, and those it should hold afterwards.
template <bool kTrim>
__device__ __forceinline__ void pages_of(const PagesP& p, int b, int& held, int& need) {
  held = imin(imax(p.held[b], 0), p.width);
  const int cached = clamp_len(p.lens[b]), fresh = kTrim ? 0 : imin(imax(p.new_lens[b], 0), p.N);
  need = imin((cached + fresh + p.page - 1) / p.page, p.width);
}

// Positions and ancestors of the new tokens, token by token.  Parents come before their children, so the walk from a token up to its root
// meets the words of its bit row from the last to the first and ends after at most i steps.
__device__ __forceinline__ void place_tokens(const PagesP& p, long long first, long long step) {
  const long long items = (long long)p.B * p.N;
  for (long long at = first; at < items; at += step) {
    const int b = (int)(at / p.N), i = (int)(at - (long long)b * p.N);
    const int cached = clamp_len(p.lens[b]), fresh = imin(imax(p.new_lens[b], 0), p.N);
    const bool real = i < fresh;
    int depth = i;
    if (p.parents != nullptr) {
      const int* parent = p.parents + (long long)b * p.N;
      unsigned* bits = reinterpret_cast<unsigned*>(p.ancestors) + at * p.words;
      int w = p.words - 1;
      unsigned word = 0;
      depth = -1;
      for (int node = real ? i : -1; node >= 0;) {
        const int up = parent[node];
        for (; w > (node >> 5); --w, word = 0) bits[w] = word;
        word |= 1u << (node & 31);
        ++depth;
        node = up < node ? up : -1;
      }
      for (; w >= 0; --w, word = 0) bits[w] = word;
    }
    p.positions[at] = real ? cached + depth : 0;
  }
}

template <bool kTrim>
__global__ void __launch_bounds__(kPageThreads) pages_kernel(PagesP p, int ctas) {
  __shared__ int before[kOwnRequests];  // off_b or r_b of this CTA's requests
  const int rank = (int)blockIdx.x;
  if (!kTrim && rank >= ctas) {  // another cluster than the one with the pages
    place_tokens(p, (long long)(rank - ctas) * kPageThreads + threadIdx.x, (long long)((int)gridDim.x - ctas) * kPageThreads);
    return;
  }
  const int per = (p.B + ctas - 1) / ctas, b0 = imin(rank * per, p.B), b1 = imin(b0 + per, p.B);
  const int n_free = imin(imax(*p.n_free, 0), p.num_pages);
  int sum = 0;
  // trim needs the sum over all requests in every CTA, reserve in the last one, which writes n_free
  const int until = (kTrim || rank == ctas - 1) ? p.B : b1;
  for (int base = 0; base < until; base += kPageThreads) {
    const int b = base + (int)threadIdx.x;
    int held = 0, need = 0, v = 0;
    if (b < p.B) {
      pages_of<kTrim>(p, b, held, need);
      v = kTrim ? imax(held - need, 0) : imax(need - held, 0);
    }
    int total;
    const int x = block_scan(v, total);
    if (b >= b0 && b < b1) before[b - b0] = sum + x;
    sum += total;
  }
  cluster_sync();  // every CTA has read `held` and `n_free`

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int b = b0 + warp; b < b1; b += kPageThreads / 32) {
    int held, need;
    pages_of<kTrim>(p, b, held, need);
    const int off = before[b - b0];
    int* row = p.table + b * p.table_sb;
    __syncwarp();  // all lanes have read held[b] and off
    if (kTrim) {
      for (int j = lane; j < held - need; j += 32) {
        const long long at = (long long)n_free + sum - 1 - (off + j);  // `held` can be nonsense
        if (at >= 0 && at < p.num_pages) p.free_pages[at] = row[need + j];
        row[need + j] = -1;
      }
      if (lane == 0) p.held[b] = imin(held, need);
    } else {
      const int got = imin(imax(need - held, 0), imax(n_free - off, 0));
      for (int j = lane; j < got; j += 32) row[held + j] = p.free_pages[n_free - 1 - (off + j)];
      if (lane == 0) {
        p.held[b] = held + got;
        before[b - b0] = p.N;  // from here on: number of the first new token without a slot (all lanes have read `off`)
      }
    }
  }
  if (rank == ctas - 1 && threadIdx.x == 0) {
    if (kTrim) {
      *p.n_free = imin(sum, p.num_pages - n_free) + n_free;
    } else {
      *p.n_free = n_free - imin(sum, n_free);
      *p.missing = imax(sum - n_free, 0);
    }
  }
  if (kTrim) return;

  __syncthreads();  // the tables' new entries are written
  const int items = (b1 - b0) * p.N;
  for (int it = threadIdx.x; it < items; it += kPageThreads) {
    const int own = it / p.N, i = it - own * p.N, b = b0 + own;
    const int cached = clamp_len(p.lens[b]), fresh = imin(imax(p.new_lens[b], 0), p.N);
    const int t = cached + i, block = t / p.page;
    int slot = -1;
    if (i < fresh && block < p.width) {
      const int page = p.table[b * p.table_sb + block];
      if (page >= 0 && page < p.num_pages) slot = page * p.page + (t - block * p.page);
    }
    p.slots[(long long)b * p.N + i] = slot;
    if (slot < 0 && i <= fresh) atomicMin(&before[own], i);
  }
  if (p.stored != nullptr) {
    __syncthreads();
    for (int own = threadIdx.x; own < b1 - b0; own += kPageThreads) p.stored[b0 + own] = before[own];
  }
  if ((int)gridDim.x == ctas) place_tokens(p, (long long)rank * kPageThreads + threadIdx.x, (long long)ctas * kPageThreads);
}

template <bool kTrim>
static int launch_pages(const PagesP& p, cudaStream_t st) {
  const long long tokens = (long long)p.B * p.N;
  const int ctas = p.B <= 64 && tokens <= 2 * kPageThreads ? 1 : kPageCtas;
  // tokens of large trees: a thread each, up to 16 clusters of them
  const int more = kTrim || ctas == 1 ? 0 : (int)((tokens + kPageCtas * kPageThreads - 1) / (kPageCtas * kPageThreads) < 16 ? (tokens + kPageCtas * kPageThreads - 1) / (kPageCtas * kPageThreads) : 16);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(ctas + more * kPageCtas));
  cfg.blockDim = dim3(kPageThreads);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, pages_kernel<kTrim>, p, ctas);
  if (e != cudaSuccess) return record_cuda_failure(e, "pages launch");
  count_launches(1);
  return CHILL_OK;
}

static int check_pages(const chill_pages_args* a, bool trim) {
  if (a == nullptr || a->B <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->table_width <= 0) return CHILL_E_INVALID;
  if (a->B > kMaxRequests || (long long)a->num_pages * a->page_size > 0x7fffffffll ||
      (long long)a->table_width * a->page_size > kMaxLen ||
      (long long)a->B * a->table_width > 0x7fffffffll)  // what the requests can hold, take or give back is summed up in 32 bits
    return CHILL_E_TOO_LARGE;
  if (!a->table || !a->held || !a->free_pages || !a->n_free || !a->lens) return CHILL_E_INVALID;
  if (a->table_stride < a->table_width && a->B > 1) return CHILL_E_INVALID;
  if (trim) return CHILL_OK;
  if (a->N <= 0 || !a->missing || !a->new_lens || !a->slots || !a->positions) return CHILL_E_INVALID;
  if ((long long)((a->B + kPageCtas - 1) / kPageCtas) * a->N > 0x7fffffffll || a->N > kMaxLen) return CHILL_E_TOO_LARGE;
  if ((a->parents == nullptr) != (a->ancestors == nullptr)) return CHILL_E_INVALID;
  return CHILL_OK;
}

static PagesP pages_params(const chill_pages_args& a, int32_t* stored) {
  PagesP p{};
  p.B = a.B; p.N = a.N; p.page = a.page_size; p.num_pages = a.num_pages; p.width = a.table_width;
  p.words = (a.N + 31) / 32;
  p.table = a.table; p.table_sb = a.table_stride;
  p.held = a.held; p.free_pages = a.free_pages; p.n_free = a.n_free; p.missing = a.missing;
  p.lens = a.lens; p.new_lens = a.new_lens; p.parents = a.parents;
  p.slots = a.slots; p.positions = a.positions; p.ancestors = a.ancestors;
  p.stored = stored;
  return p;
}

// ------------------------------------------------------------------------------------------------------ append
// Row (b, head, i) of K and V to slot slots[b][i]: a copy, bound by memory.  A thread moves one vector of K and the same one of V;
// V is 16 bytes, or one element where a layout allows no more.  2048 new tokens for each of 16 requests (262 MB read and written): 45 us,
// 5.8 TB/s of the 6.5 of a plain copy; with the vectors of two requests in flight a thread 47 us.
struct RowsP {
  int B, Hkv, N, page, num_pages, per_row, per_token;  // vectors of a row (head) and of a token
  const char *k, *v;
  char *kc, *vc;
  long long ks[4], vs[4];    // byte strides of [batch][head][token], then of a vector's channels
  long long kcs[4], vcs[4];  // byte strides of [page][head][row], then of a vector's channels
  const int* slots;
  // commit
  const int *table, *lens, *new_lens, *path, *accepted;
  long long table_sb;
  int width, A;
  int moved;  // vectors of a token that move: those of K and V, or where both are one tensor those of it
  int* out_lens;
};

template <typename V>
__global__ void __launch_bounds__(256) append_kernel(RowsP p) {
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;  // N * per_token < 2^31
  if (idx >= (unsigned)p.N * (unsigned)p.per_token) return;
  const int i = (int)(idx / (unsigned)p.per_token), rem = (int)(idx - (unsigned)i * (unsigned)p.per_token);
  const int h = rem / p.per_row, c = rem - h * p.per_row;
  const char* k = p.k + h * p.ks[1] + i * p.ks[2] + c * p.ks[3];
  const char* v = p.v + h * p.vs[1] + i * p.vs[2] + c * p.vs[3];
  char* kc = p.kc + h * p.kcs[1] + c * p.kcs[3];
  char* vc = p.vc + h * p.vcs[1] + c * p.vcs[3];
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int slot = p.slots[(long long)b * p.N + i];
    if (slot < 0 || slot >= p.num_pages * p.page) continue;
    const V x = *reinterpret_cast<const V*>(k + b * p.ks[0]), y = *reinterpret_cast<const V*>(v + b * p.vs[0]);
    const int page = slot / p.page, row = slot - page * p.page;
    *reinterpret_cast<V*>(kc + page * p.kcs[0] + row * p.kcs[2]) = x;
    *reinterpret_cast<V*>(vc + page * p.vcs[0] + row * p.vcs[2]) = y;
  }
}

// ------------------------------------------------------------------------------------------------------ commit
// Row lens[b] + path[b][j] -> row lens[b] + j for j < accepted[b].  The path increases, so path[j] >= j: no row is written before
// the rows that it is the source of have been read, as long as j runs upwards.  A thread owns one vector of every row (of K or of
// V), so no two threads meet; it reads kBatch rows before it writes them, which only reads rows earlier than the order asks for.
// A row without a page was never stored, so the path ends there: a CTA of its own, a lane for each token of the path, works out how long it is
// (by the thread of the first vector, on its way, it took the call 2 us longer: 9 of 64 drafts for 128 requests, 22.6 us with the append).
constexpr int kBatch = 8;

template <typename V>
__global__ void __launch_bounds__(128) commit_kernel(RowsP p) {
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int cached = clamp_len(p.lens[b]), fresh = imin(imax(p.new_lens[b], 0), p.N);
    const int take = imin(imin(imax(p.accepted[b], 0), p.A), fresh);
    const int* table = p.table + b * p.table_sb;
    const int* path = p.path + (long long)b * p.A;
    auto page_of = [&](int t) -> int {  // -1 where there is none
      const int block = t / p.page, page = block < p.width ? table[block] : -1;
      return page < p.num_pages ? imax(page, -1) : -1;
    };
    if (blockIdx.x == gridDim.x - 1) {
      if (threadIdx.x >= 32) continue;
      int kept = take;
      for (int j0 = 0; j0 < take; j0 += 32) {
        const int j = j0 + (int)threadIdx.x, from = j < take ? path[j] : 0;
        const bool moves = from > j && from < fresh;
        const unsigned lost = __ballot_sync(0xffffffffu, j < take && (page_of(cached + j) < 0 || (moves && page_of(cached + from) < 0)));
        if (lost == 0) continue;
        kept = j0 + __ffs(lost) - 1;
        break;
      }
      if (threadIdx.x == 0) p.out_lens[b] = cached + kept;
      continue;
    }
    const int idx = blockIdx.x * 128 + threadIdx.x;
    if (idx >= p.moved) continue;
    const bool is_v = idx >= p.per_token;
    const int rem = is_v ? idx - p.per_token : idx, h = rem / p.per_row, c = rem - h * p.per_row;
    const long long* st = is_v ? p.vcs : p.kcs;
    char* base = (is_v ? p.vc : p.kc) + h * st[1] + c * st[3];
    auto row_of = [&](int t) -> char* {  // nullptr where there is no page
      const int page = page_of(t);
      return page < 0 ? nullptr : base + page * st[0] + t % p.page * st[2];
    };
    int from[kBatch];  // asked for before it is known how many count: one trip to memory less
#pragma unroll
    for (int u = 0; u < kBatch; ++u) from[u] = u < p.A ? path[u] : 0;
    for (int j0 = 0; j0 < take; j0 += kBatch) {
      if (j0 != 0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) from[u] = j0 + u < take ? path[j0 + u] : 0;
      }
      const char* src[kBatch];
      char* dst[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {  // in place already, or not a drafted token: no move
        const bool moves = j0 + u < take && from[u] > j0 + u && from[u] < fresh;
        src[u] = moves ? row_of(cached + from[u]) : nullptr;
        dst[u] = moves ? row_of(cached + j0 + u) : nullptr;
      }
      V x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (src[u] != nullptr) x[u] = *reinterpret_cast<const V*>(src[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (src[u] != nullptr && dst[u] != nullptr) *reinterpret_cast<V*>(dst[u]) = x[u];
    }
  }
}

static bool vec16(const void* p, const int64_t* st, int es) {
  if (st[3] != 1 || reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int d = 0; d < 3; ++d)
    if ((st[d] * es) % 16 != 0) return false;
  return true;
}

static void byte_strides(long long* to, const int64_t* st, int es, int vec) {
  for (int d = 0; d < 3; ++d) to[d] = (long long)st[d] * es;
  to[3] = vec == 1 ? (long long)st[3] * es : 16;
}

static int check_rows(const chill_cache_rows_args* a) {
  if (a == nullptr || a->B <= 0 || a->H_kv <= 0 || a->N <= 0 || a->D <= 0 || a->num_pages <= 0 || a->page_size <= 0) return CHILL_E_INVALID;
  if (a->dtype != CHILL_F32 && a->dtype != CHILL_F16 && a->dtype != CHILL_BF16) return CHILL_E_UNSUPPORTED;
  if ((long long)a->num_pages * a->page_size > 0x7fffffffll || a->N > kMaxLen || a->B > kMaxRequests || (long long)a->H_kv * a->D > (1 << 28)) return CHILL_E_TOO_LARGE;
  if (!a->k_cache || !a->v_cache) return CHILL_E_INVALID;
  return CHILL_OK;
}

}  // namespace cache
}  // namespace chill

using namespace chill;
using namespace chill::cache;

extern "C" {

int chill_pages_reserve_stored(const chill_pages_args* a, int32_t* stored, void* stream) {
  int st = check_pages(a, false);
  if (st == CHILL_OK && stored != nullptr)  // written while CTAs read and write the others
    for (const int32_t* other : {a->lens, a->new_lens, a->parents, (const int32_t*)a->table, (const int32_t*)a->held, (const int32_t*)a->free_pages, (const int32_t*)a->n_free,
                                 (const int32_t*)a->missing, (const int32_t*)a->slots, (const int32_t*)a->positions, (const int32_t*)a->ancestors})
      if (stored == other) st = CHILL_E_INVALID;
  return st != CHILL_OK ? st : launch_pages<false>(pages_params(*a, stored), (cudaStream_t)stream);
}

int chill_pages_reserve(const chill_pages_args* a, void* stream) { return chill_pages_reserve_stored(a, nullptr, stream); }

int chill_pages_trim(const chill_pages_args* a, void* stream) {
  const int st = check_pages(a, true);
  return st != CHILL_OK ? st : launch_pages<true>(pages_params(*a, nullptr), (cudaStream_t)stream);
}

int chill_cache_append(const chill_cache_rows_args* a, void* stream) {
  int st = check_rows(a);
  if (st != CHILL_OK) return st;
  if (!a->k || !a->v || !a->slots) return CHILL_E_INVALID;
  const int es = a->dtype == CHILL_F32 ? 4 : 2;
  const bool wide = a->D * es % 16 == 0 && vec16(a->k, a->k_strides, es) && vec16(a->v, a->v_strides, es) &&
                    vec16(a->k_cache, a->k_cache_strides, es) && vec16(a->v_cache, a->v_cache_strides, es);
  const int vec = wide ? 16 / es : 1;
  RowsP p{};
  p.B = a->B; p.Hkv = a->H_kv; p.N = a->N; p.page = a->page_size; p.num_pages = a->num_pages;
  p.per_row = a->D / vec; p.per_token = p.per_row * a->H_kv;
  p.k = (const char*)a->k; p.v = (const char*)a->v; p.kc = (char*)a->k_cache; p.vc = (char*)a->v_cache;
  byte_strides(p.ks, a->k_strides, es, vec); byte_strides(p.vs, a->v_strides, es, vec);
  byte_strides(p.kcs, a->k_cache_strides, es, vec); byte_strides(p.vcs, a->v_cache_strides, es, vec);
  p.slots = a->slots;
  const long long vectors = (long long)p.N * p.per_token;
  if (vectors > 0x7fffff00ll) return CHILL_E_TOO_LARGE;
  const long long blocks = (vectors + 255) / 256;
  const dim3 grid((unsigned)blocks, (unsigned)imin(a->B, 65535));
  if (wide) append_kernel<uint4><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else if (es == 4) append_kernel<uint32_t><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  else append_kernel<uint16_t><<<grid, 256, 0, (cudaStream_t)stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_cuda_failure(e, "append launch");
  count_launches(1);
  return CHILL_OK;
}

int chill_cache_commit(const chill_cache_rows_args* a, void* stream) {
  int st = check_rows(a);
  if (st != CHILL_OK) return st;
  if (!a->table || !a->lens || !a->new_lens || !a->path || !a->accepted || !a->out_lens || a->table_width <= 0 || a->A <= 0) return CHILL_E_INVALID;
  if (a->out_lens == a->lens) return CHILL_E_INVALID;  // a request has several CTAs, all of them read its length
  if ((long long)a->table_width * a->page_size > kMaxLen) return CHILL_E_TOO_LARGE;
  const int es = a->dtype == CHILL_F32 ? 4 : 2;
  const bool wide = a->D * es % 16 == 0 && vec16(a->k_cache, a->k_cache_strides, es) && vec16(a->v_cache, a->v_cache_strides, es);
  const int vec = wide ? 16 / es : 1;
  RowsP p{};
  p.B = a->B; p.Hkv = a->H_kv; p.N = a->N; p.page = a->page_size; p.num_pages = a->num_pages;
  p.per_row = a->D / vec; p.per_token = p.per_row * a->H_kv;
  p.kc = (char*)a->k_cache; p.vc = (char*)a->v_cache;
  byte_strides(p.kcs, a->k_cache_strides, es, vec); byte_strides(p.vcs, a->v_cache_strides, es, vec);
  p.table = a->table; p.table_sb = a->table_stride; p.width = a->table_width;
  p.lens = a->lens; p.new_lens = a->new_lens; p.path = a->path; p.accepted = a->accepted; p.A = a->A; p.out_lens = a->out_lens;
  // K and V in one tensor: each row moves once (two threads that move it one after the other would read what the other has written)
  bool one = a->k_cache == a->v_cache;
  for (int d = 0; d < 4 && one; ++d)
    if (a->k_cache_strides[d] != a->v_cache_strides[d]) return CHILL_E_INVALID;
  p.moved = (one ? 1 : 2) * p.per_token;
  const dim3 grid((unsigned)((p.moved + 127) / 128 + 1), (unsigned)imin(a->B, 65535));
  if (wide) commit_kernel<uint4><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  else if (es == 4) commit_kernel<uint32_t><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  else commit_kernel<uint16_t><<<grid, 128, 0, (cudaStream_t)stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return record_cuda_failure(e, "commit launch");
  count_launches(1);
  return CHILL_OK;
}

}  // extern "C"
