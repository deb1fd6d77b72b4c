/*
 * chill_cache.h - C ABI of the operators that serve a model from a paged cache (libchill_cache_b200.so; kernels for sm_100a).
 *
 * Conventions, status codes, element types, masks and flags are those of chill_b200.h: plain device pointers and element strides, work
 * is enqueued on the given stream of the current device, nothing allocates, synchronises or keeps state between calls (but for the
 * record of which kernels had their shared-memory limit raised, and counters), 0 on success and a negative CHILL_E_* code otherwise.
 */
#ifndef CHILL_CACHE_H_
#define CHILL_CACHE_H_

#include "chill_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHILL_CACHE_ABI_VERSION 1

/* ------------------------------------------------------------------------------------------------------------------
 * Serving from a paged cache (no counterpart in the reference, which attends whole sequences only).
 *
 * Keys and values of request b live in pages of page_size rows: the row of position t is row t % page_size of page
 * table[b * table_stride + t / page_size]; a table entry outside [0, num_pages) is no page, and its keys are not there.  Cache
 * tensors are indexed [page][kv head][row][channel], k_cache_strides / v_cache_strides in elements.  A step adds new_lens[b] tokens
 * (clamped to [0, N]) behind the lens[b] that are cached: one each, a chunk, or a tree of drafted tokens.  All of it is read on the
 * GPU, nothing here synchronises, and every call can be captured into a graph and replayed with other lengths.  Calls that use
 * the same pages are ordered by the caller (one stream, or events).  All integer arrays are int32, device, contiguous unless a stride
 * is given.  Sizes: B <= 65535, num_pages * page_size < 2^31, table_width * page_size <= 2^29, for reserve and trim
 * B * table_width < 2^31 (CHILL_E_TOO_LARGE). */

typedef struct chill_pages_args {
  int32_t B, N;  /* requests; most new tokens of a request */
  int32_t page_size, num_pages, table_width;
  int32_t reserved;
  int32_t* table; /* [B][table_width], rows table_stride apart */
  int64_t table_stride;
  int32_t* held;       /* [B]: pages of each request */
  int32_t* free_pages; /* [num_pages]: a stack; what lies at n_free and above is left over */
  int32_t* n_free;     /* [1] */
  int32_t* missing;    /* [1], reserve: pages that were wanted and not there */
  const int32_t *lens, *new_lens; /* [B]; trim does not look at new_lens */
  const int32_t* parents;         /* reserve, [B][N] or NULL: parent of each new token of a tree, by number; a value outside
                                   * [0, own number) is the last cached token */
  int32_t *slots, *positions;     /* reserve, [B][N]: page * page_size + row (-1: not a token, or no page); position (0: not a token) */
  int32_t* ancestors;             /* reserve, [B][N][(N + 31) / 32], with parents: bit j of row i: token j is token i or above it */
} chill_pages_args;

/* Pages for lens[b] + new_lens[b] tokens of every request, from the top of the stack, requests in order; then slots, positions
 * (lens[b] + depth; without parents lens[b] + number) and ancestors of the new tokens.  Pages that a request holds beyond
 * that stay its own.  Where pages run out, or a table is full, the tokens without one get slot -1. */
int chill_pages_reserve(const chill_pages_args* a, void* stream);
/* The same, and in stored[b] (may be NULL; an array of its own) how many of a request's new tokens got a slot: the first so many.  Where there was a shortage only these
 * may be counted in lens afterwards; the others' rows are never written, and a page that turns up for them later holds its former owner's. */
int chill_pages_reserve_stored(const chill_pages_args* a, int32_t* stored, void* stream);
/* Pages behind lens[b] tokens go back to the stack (lens[b] = 0: all), their table entries become -1.  The inverse of reserve: the
 * pages come back in the order in which reserving them again takes them. */
int chill_pages_trim(const chill_pages_args* a, void* stream);

typedef struct chill_cache_rows_args {
  int32_t B, H_kv, N, D, dtype;
  int32_t page_size, num_pages, table_width, A;
  int32_t reserved;
  void *k_cache, *v_cache;
  int64_t k_cache_strides[4], v_cache_strides[4];
  const void *k, *v; /* append: [batch][kv head][token][channel] */
  int64_t k_strides[4], v_strides[4];
  const int32_t* slots; /* append: [B][N] */
  const int32_t* table; /* commit, and the rest */
  int64_t table_stride;
  const int32_t *lens, *new_lens; /* [B] */
  const int32_t* path;            /* [B][A]: numbers of the accepted tokens, increasing */
  const int32_t* accepted;        /* [B]: how many of them, clamped to [0, min(A, new_lens[b])] */
  int32_t* out_lens;              /* [B]: lens[b] + accepted[b], as far as these have a page; not lens itself */
} chill_cache_rows_args;

/* Row (b, head, i) of k and v goes to slot slots[b][i] of the caches; slots outside the cache are skipped. */
int chill_cache_append(const chill_cache_rows_args* a, void* stream);
/* The accepted path of every tree becomes contiguous: for j < accepted[b], row lens[b] + path[b][j] is copied to row lens[b] + j
 * (path[b][j] <= j: it stays as it is).  The path ends before the first token without a page.  k_cache and v_cache may be one tensor (then with
 * one set of strides), but not overlap in another way. */
int chill_cache_commit(const chill_cache_rows_args* a, void* stream);

/* O = softmax(mask(Q K^T * sm_scale)) V of the new tokens over the cached and the new keys, and its LSE (log2 units).  The rows of
 * the new tokens must be in the cache (chill_cache_append).  Token i of request b, at position p = positions[b][i] (a chain: lens[b] + i),
 * sees cached key t iff mask(p, t), and new key j iff mask(p, positions[b][j]) and, in a tree, j is an ancestor of i or i itself.
 * The mask functor gets lens[b] + new_lens[b] as the sequence length.  A token that sees nothing: O = 0, LSE = -inf; rows at and
 * behind new_lens[b]: O = 0, LSE = 0. */
typedef struct chill_cached_args {
  chill_mask_desc mask;
  int32_t B, H, H_kv, N, D, dtype;
  int32_t page_size, num_pages, table_width;
  float sm_scale;
  uint32_t flags; /* CHILL_FLAG_FORCE_GENERIC */
  int32_t reserved;
  const void *q, *k_cache, *v_cache;
  void* o;
  float* lse; /* may be NULL */
  int64_t q_strides[4], k_cache_strides[4], v_cache_strides[4], o_strides[4];
  int64_t lse_strides[3];
  const int32_t* table;
  int64_t table_stride;
  const int32_t *lens, *new_lens;
  const int32_t *positions, *ancestors; /* of chill_pages_reserve; ancestors NULL: a chain, positions are not looked at */
  void* workspace;                      /* chill_cached_workspace_bytes() bytes, 256-byte aligned; one for each call that can overlap */
  size_t workspace_bytes;
} chill_cached_args;
size_t chill_cached_workspace_bytes(const chill_cached_args* a);
int chill_cached_fwd(const chill_cached_args* a, void* stream);
/* Which kernel chill_cached_fwd would launch (host-only; pointers are looked at for their alignment), or a negative status. */
#define CHILL_CACHED_CUDA_CORES 0 /* fp32, and what the others can not take */
#define CHILL_CACHED_ROWS 1       /* 16-bit, up to 32 rows (N * H / H_kv) of a kv head, 16 above head dim 128, and queries that the tiles can not take */
#define CHILL_CACHED_TILES 2      /* 16-bit, tiles of 128 rows */
int chill_cached_kernel(const chill_cached_args* a);

/* As chill_read_device_status (0: no kernel of this library gave up a wait since the last look; a call whose kernel did has incomplete results), chill_launch_count and chill_last_cuda_error, for this library. */
int chill_cache_read_device_status(void);
unsigned long long chill_cache_launch_count(void);
const char* chill_cache_last_cuda_error(void);
int chill_cache_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CHILL_CACHE_H_ */
