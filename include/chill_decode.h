/*
 * chill_decode.h - C ABI of the operators around attention (libchill_decode_b200.so; kernels for sm_100a): rotary positions, the selection
 * of a beam search, pages that several requests share, copies and compaction of pages.
 *
 * Conventions, status codes and element types are those of chill_b200.h, pages, tables and caches those of chill_cache.h: plain device
 * pointers and element strides, work is enqueued on the given stream of the current device, nothing allocates, synchronises or keeps
 * state between calls (but for the record of which kernels had their shared-memory limit raised, and counters), 0 on success and a negative
 * CHILL_E_* code otherwise.  Every call can be captured into a graph and replayed.  The reference has no counterpart.
 */
#ifndef CHILL_DECODE_H_
#define CHILL_DECODE_H_

#include "chill_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CHILL_DECODE_ABI_VERSION 1

/* ------------------------------------------------------------------------------------------------------------------
 * Rotary positions.  Pair i of a row at positions p is turned by the angle p[axes[i]] * inv_freq[i]:
 *     y1 = x1 cos a - x2 sin a,  y2 = x2 cos a + x1 sin a          (inverse: the angle -a, which is the backward)
 * Pair i is channels (i, i + pairs), or with interleaved (2 i, 2 i + 1); channels from 2 * pairs on stay as they are.  Angles are worked out in
 * 64 bits, the rest in fp32, and results are rounded once. */
typedef struct chill_rotate_args {
  int32_t B, H, H_kv, L, D, dtype;
  int32_t pairs;       /* 1 <= pairs, 2 * pairs <= D */
  int32_t n_axes;      /* rows of positions */
  int32_t interleaved; /* 0 or 1 */
  int32_t inverse;     /* 0 or 1; chill_rotate_append: 0 */
  const float* inv_freq;         /* [pairs], radians a position */
  const int32_t* axes;           /* [pairs], row of positions that turns a pair (clamped to [0, n_axes)), or NULL: the first one */
  const int32_t* positions;      /* [axis][batch][token] */
  int64_t position_strides[3];
  const void *q, *k;             /* [batch][head][token][channel]; q with H heads, k with H_kv; either may be NULL in chill_rotate, with its result */
  int64_t q_strides[4], k_strides[4];
  void *q_out, *k_out;           /* results; neither may overlap an input.  chill_rotate_append does not look at k_out */
  int64_t q_out_strides[4], k_out_strides[4];
  /* chill_rotate_append: row (b, head, i) of k, turned, and of v, as it is, go to slot slots[b][i] of the caches ([page][kv head][row][channel]);
   * slots outside the caches are skipped */
  const void* v;
  int64_t v_strides[4];
  void *k_cache, *v_cache;
  int64_t k_cache_strides[4], v_cache_strides[4];
  const int32_t* slots; /* [B][L] */
  int32_t num_pages, page_size;
} chill_rotate_args;
/* Sizes: B * L * D < 2^31, num_pages * page_size < 2^31 (CHILL_E_TOO_LARGE). */
int chill_rotate(const chill_rotate_args* a, void* stream);
int chill_rotate_append(const chill_rotate_args* a, void* stream);

/* ------------------------------------------------------------------------------------------------------------------
 * Selection over beams and vocabulary.  Candidate (k, v) of group g: c = scores[g][k] + x - log sum exp x', x = logits[g * K + k][v], the sum over the
 * row; -inf where the logit or the beam's score is -inf.  A finished beam has one candidate, (k, end_token) with c = scores[g][k], and its
 * logits are not looked at.  The M candidates of the largest c in descending order, of equal ones the lowest k, then the largest x (64 bits round c, and neighbouring
 * logits may share it), then the lowest v.  c is worked out, ranked and kept in 64 bits until it is written, but the terms of its sum are fp32 exponentials, up to 32 of them
 * a thread added in fp32: the logarithm is good to 1e-7 in ordinary rows, and to 1e-5 where a row's maximum rises again and again along it (measured: 6e-8, 3e-6).  Candidates of one beam are in the exact
 * order of their logits; those of different beams that are nearer than that may change places.  Equal rows (not permutations of one another) have equal sums, bit
 * for bit.  NaN counts as largest: a NaN or +inf among a row's logits, or a NaN as score, makes all its candidates NaN, but for those of -inf; these, and those of a beam of score
 * +inf, are alike, the lowest v first. */
#define CHILL_SELECT_MAX 64 /* beams of a group, and candidates that are kept */
typedef struct chill_select_args {
  int32_t G, K, M, dtype;
  int64_t V;               /* <= 2^26 */
  const void* logits;      /* [G * K][V], rows row_stride elements apart, their elements adjacent */
  int64_t row_stride;
  const float* scores;     /* [G][K], logarithms; -inf: no such beam */
  const uint8_t* finished; /* [G][K], not zero: finished; or NULL */
  int64_t end_token;       /* in [0, V), looked at with finished */
  float* out_scores;       /* [G][M] */
  int32_t* out_rows;       /* [G][M], g * K + k */
  int32_t* out_tokens;     /* [G][M] */
  void* workspace;         /* chill_select_workspace_bytes() bytes, 16-byte aligned; one for each call that can overlap */
  size_t workspace_bytes;
} chill_select_args;
/* 1 <= K, M <= CHILL_SELECT_MAX, M <= K * V, G * K <= 65535. */
size_t chill_select_workspace_bytes(const chill_select_args* a); /* from G, K, M, V, dtype and the current device alone */
int chill_beam_select(const chill_select_args* a, void* stream);

/* ------------------------------------------------------------------------------------------------------------------
 * Pages that several requests hold.  shared[page] counts the holders beyond one: 0 for a page that one request holds and for a free one, so that
 * chill_pages_reserve hands out pages as ever.  Tables, held, free_pages and n_free are those of chill_pages_args.  Sizes: num_pages <= 2^30,
 * num_pages * page_size < 2^31, table_width * page_size <= 2^29, B <= 65535, B * table_width <= 2^31 - 16 (CHILL_E_TOO_LARGE). */
typedef struct chill_share_args {
  int32_t B, page_size, num_pages, table_width;
  int32_t* table; /* [B][table_width], rows table_stride apart */
  int64_t table_stride;
  int32_t* held;       /* [B] */
  int32_t* free_pages; /* [num_pages] */
  int32_t* n_free;     /* [1] */
  int32_t* shared;     /* [num_pages]; chill_pages_compact: may be NULL */
  const int32_t* lens; /* [B]; not chill_pages_compact */
  /* chill_pages_fork */
  int32_t* missing;       /* [1] */
  const int32_t* parents; /* [B] */
  int32_t* out_lens;      /* [B] */
  /* chill_pages_fork ([B]) and chill_pages_compact ([max(num_pages / 2, 1)]): what is to be copied, *count orders from the front on, behind
   * them -1, -1, 0 */
  int32_t *source, *target, *rows;
  int32_t* count;  /* [1] */
  void* workspace; /* chill_share_workspace_bytes() bytes, 16-byte aligned; one for each call that can overlap */
  size_t workspace_bytes;
} chill_share_args;
/* Row b takes over what row parents[b] holds of its lens[parents[b]] tokens (a parent outside [0, B): nothing).  Whole pages are shared.  A page that is
 * only begun goes to the first child, if nobody else holds it; every other child gets a page of its own from the stack and an order to copy the rows
 * into it.  Where the stack runs out the child keeps its whole pages only; missing says how many pages were short.  Pages that nobody holds any more go back
 * to the stack: in the order of the rows and blocks that held them first, the first on top.  out_lens: tokens of each row now.  B <= 8192. */
int chill_pages_fork(const chill_share_args* a, void* stream);
/* chill_pages_trim for pages that may be shared: those behind lens[b] tokens are let go of, and go back to the stack when nobody else holds them. */
int chill_pages_trim_shared(const chill_share_args* a, void* stream);
/* Pages in use move to the bottom of the pool: with U of them, the highest used page goes to the lowest free one below U, and so on.  Tables, shared and
 * the stack (lowest page on top) follow; the caches are moved by chill_cache_copy. */
int chill_pages_compact(const chill_share_args* a, void* stream);
/* From B, num_pages and table_width alone. */
size_t chill_share_workspace_bytes(const chill_share_args* a);

/* The first rows[i] rows of page source[i] are copied to page target[i], for i < *count, in both caches and all layers.  Orders with a page outside
 * [0, num_pages) are skipped.  No target may be a source or target of another order. */
typedef struct chill_copy_args {
  int32_t layers, num_pages, H_kv, page_size, D, dtype;
  void *k_cache, *v_cache;                        /* [layer][page][kv head][row][channel] */
  int64_t k_cache_strides[5], v_cache_strides[5];
  const int32_t *source, *target, *rows, *count; /* rows: clamped to [0, page_size]; *count: clamped to [0, orders] */
  int32_t orders;                                 /* length of source, target and rows */
  int32_t reserved;
} chill_copy_args;
int chill_cache_copy(const chill_copy_args* a, void* stream);

/* As chill_launch_count and chill_last_cuda_error, for this library. */
unsigned long long chill_decode_launch_count(void);
const char* chill_decode_last_cuda_error(void);
int chill_decode_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CHILL_DECODE_H_ */
