// C ABI of the paged cache (include/chill_cache.h): attention, i.e. checks of the arguments, choice of the kernel, workspace, TMA
// descriptors, launch; and the library's records.  The other operators are in cache_pages.cu.
#include <cuda.h>
#include <cuda_runtime.h>

#include "abi_common.cuh"
#include "cache_common.cuh"
#include "cache_launch.h"
#include "chill_cache.h"
#include "tc_launch.h"

namespace chill {

int record_cuda_failure(cudaError_t e, const char* what) { return cuda_fail(e, what); }  // for cache_pages.cu
void count_launches(int n) { g_launches += n; }

namespace cache {

static int check_cached(const chill_cached_args* a, bool pointers) {
  if (a == nullptr || a->B <= 0 || a->H <= 0 || a->H_kv <= 0 || a->N <= 0 || a->D <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->table_width <= 0)
    return CHILL_E_INVALID;
  if (a->H % a->H_kv != 0) return CHILL_E_INVALID;
  if (a->dtype != CHILL_F32 && a->dtype != CHILL_F16 && a->dtype != CHILL_BF16) return CHILL_E_UNSUPPORTED;
  if (a->D > kMaxD || a->D % 16 != 0) return CHILL_E_UNSUPPORTED;
  if (a->B > 65535 || a->H > 65535 || a->N > kMaxLen / 2 || (long long)a->N * (a->H / a->H_kv) > kMaxLen ||
      (long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->table_width * a->page_size > kMaxLen)
    return CHILL_E_TOO_LARGE;
  if (!(a->sm_scale > 0.f) || a->sm_scale > 2e38f) return CHILL_E_INVALID;  // times log2(e) it stays finite
  const int st = check_mask(a->mask);
  if (st != CHILL_OK) return st;
  if (!pointers) return CHILL_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->o || !a->table || !a->lens || !a->new_lens) return CHILL_E_INVALID;
  if (a->ancestors != nullptr && a->positions == nullptr) return CHILL_E_INVALID;
  return CHILL_OK;
}

// Rows of a TMA box: the largest of 64, 32, 16, 8 that divides the page (a box lies in one page, and starts at a multiple of the
// 8 rows after which the swizzle repeats); 0: no box.
static int box_rows(int page) {
  for (int box = kKeyTile; box >= 8; box /= 2)
    if (page % box == 0) return box;
  return 0;
}

// Rows of a tile of the kernel for many rows: as many whole tokens as 128 rows hold (0: a token has more).
static int tile_rows(int G) { return G <= kTileRows ? kTileRows / G * G : 0; }

// CHILL_CACHED_*: few rows go through mma.sync, which reads the keys once for all of them, many through tiles of 128 rows.
static int cached_kernel(const chill_cached_args& a) {
  if (a.dtype == CHILL_F32 || (a.flags & CHILL_FLAG_FORCE_GENERIC) || box_rows(a.page_size) == 0) return CHILL_CACHED_CUDA_CORES;
  const size_t es = esize(a.dtype);
  if (!tma_ok(a.k_cache, a.k_cache_strides, a.num_pages, a.H_kv, a.page_size, es) || !tma_ok(a.v_cache, a.v_cache_strides, a.num_pages, a.H_kv, a.page_size, es))
    return CHILL_CACHED_CUDA_CORES;
  const int G = a.H / a.H_kv;
  if ((long long)a.N * G <= (a.D <= 128 ? 32 : 16) || tile_rows(G) == 0 || !tma_ok(a.q, a.q_strides, a.B, a.H, a.N, es)) return CHILL_CACHED_ROWS;
  return CHILL_CACHED_TILES;
}

// Kernel, tiles, CTAs and workspace of a call, from the sizes that the host knows.
struct Plan {
  int kernel, rows, row_tiles, grid, pad, min_share, tail_shares;
  bool scan;   // prefix sums by a launch of their own
  bool whole;  // CTAs take whole units
  size_t queue, seams, cum, ml, o, bytes;
};

// What a CTA spends on a unit beside its tiles (Q, the parts of O, the next piece's start), in tiles.  Kernel for few rows: 0 / 2 / 4 tiles
// 184.5 / 182.3 / 183.4 us (64 requests of up to 8192 tokens, one new each), 48.5 / 46.9 / 54.5 us (24 drafts each for 32 requests, window
// of 1024).  Kernel for many rows: 0 / 3 / 5 / 6 / 7 / 10 tiles 106.4 / 99.1 / 94.2 / 92.3 / 92.7 / 94.6 us (64 drafts for 16 requests), 437 / 418 /
// 411 / 407 / 403 to 428 / 408 to 438 us (1024 new tokens for 4 requests).
constexpr int kRowsPad = 2, kTilesPad = 6;

// Keys a token can see at most in a table of `keys` (looked at for 32 positions: what is chosen by it is a matter of time alone).
template <class M>
static long long widest(const MaskArgs& margs, int keys) {
  long long most = 0;
  for (int i = 0; i < 32; ++i) {
    int lo, hi;
    M::k_range_for_q((int)((long long)(keys - 1) * i / 31), keys, margs, lo, hi);
    lo = imax(lo, 0);
    hi = imin(hi, keys - 1);
    most = hi - lo + 1 > most ? hi - lo + 1 : most;
  }
  return most;
}

static int make_plan(const chill_cached_args& a, Plan& c) {
  const int G = a.H / a.H_kv, sms = sm_count();
  const long long group_rows = (long long)a.N * G;
  c.kernel = cached_kernel(a);
  c.min_share = 2;
  c.pad = 0;
  c.tail_shares = 0;
  const long long keys = (long long)a.table_width * a.page_size;
  // what a unit can have to do, by the size of the table and the mask
  long long seen = keys;
  CHILL_MASK_SWITCH_OR(a.mask.id, (seen = widest<MaskT>(to_mask_args(a.mask, (long long)kMaxLen), (int)keys)), )
  seen = seen + a.N < keys ? seen + a.N : keys;
  // A few tiles: one launch and no sum, whatever the lengths (2 requests of 300 cached tokens, fp32: 10 us; cut in shares, with the kernel
  // that joins them, 23 us)
  c.whole = seen <= 8 * kKeyTile;
  if (c.kernel == CHILL_CACHED_CUDA_CORES) {
    // Rows in tiles of 4 where that is faster than larger ones with more work in shared memory.  Whole units: while the SMs have few of them, up
    // to about six tiles of 4 each (24 rows, 32 / 512 units: 13.5 / 109 us, in tiles of 32 rows 38.8 / 62.8; 8 rows, 408 units: 51 / 75).  Shares: 5 to
    // 8 rows of 65 to 128 channels, though keys are read twice (one token for 16 requests of 8000, 8 heads a kv head: 118 us, in tiles of 8
    // rows 148; of 64 channels 70.5 / 68, of 256 55 / 52).
    const long long fours = (long long)a.B * a.H_kv * ((group_rows + 3) / 4);
    const bool quads = c.whole ? fours <= 6 * sms : (group_rows <= 8 && a.D > 64 && a.D <= 128);
    c.rows = group_rows <= 2 ? 2 : (group_rows <= 4 || quads ? 4 : (group_rows <= 8 ? 8 : (group_rows <= 16 ? 16 : 32)));
    c.grid = sms * (c.rows < 8 ? 4 : (a.D <= 64 ? 4 : (a.D <= 128 ? 2 : 1)));
    if (c.rows < 8) c.tail_shares = c.grid;  // 16 rows and more: 1194 us with small shares, 1136 without (500 new tokens for 2 requests)
  } else if (c.kernel == CHILL_CACHED_ROWS) {
    c.rows = group_rows <= 16 || a.D > 128 ? 16 : 32;
    c.grid = sms * rows_ctas(a.D, c.rows);
    c.tail_shares = 2 * c.grid;
    c.pad = kRowsPad;
  } else {
    const int half = tile_rows(G);
    const bool two = a.D <= 128 && group_rows > half;
    c.rows = two ? 2 * half : half;
    c.pad = kTilesPad;
    c.grid = sms * (a.D <= 128 ? 2 : 1) / (two ? 2 : 1);
  }
  const long long row_tiles = (group_rows + c.rows - 1) / c.rows, entries = (long long)a.B * row_tiles;
  if (entries * a.H_kv * (keys / kKeyTile + 8) > 0x7fffffffll) return CHILL_E_TOO_LARGE;
  c.row_tiles = (int)row_tiles;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  if (c.whole) {
    c.grid = entries * a.H_kv < c.grid ? (int)(entries * a.H_kv) : c.grid;
    c.tail_shares = 0;
  }
  // small shares only where there can be so many keys
  if (entries * a.H_kv * (seen / kKeyTile + 1) < (long long)kTailFrom * c.grid) c.tail_shares = 0;
  c.scan = !c.whole && entries > kScanEntries;
  const int shares = c.grid + c.tail_shares;
  c.queue = 0;
  c.seams = c.queue + 256;
  c.cum = c.seams + up((size_t)shares * sizeof(Seam));
  c.ml = c.cum + (c.scan ? up((size_t)(entries + 1) * 4) : 0);
  c.o = c.ml + up((size_t)2 * shares * c.rows * sizeof(float2));
  c.bytes = c.o + up((size_t)2 * shares * c.rows * a.D * sizeof(float));
  return CHILL_OK;
}

// Q by whole tokens: channels, heads of a group, tokens, kv heads, requests; a box is 64 channels of `tokens` tokens' rows of a group.
static int make_q_map(CUtensorMap* m, const chill_cached_args& a, int tokens) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return cuda_fail(cudaErrorUnknown, "cuTensorMapEncodeTiled entry point not available");
  const int G = a.H / a.H_kv;
  const cuuint64_t es = esize(a.dtype), any = 16;  // strides of dimensions of size one are not looked at
  cuuint64_t dims[5] = {(cuuint64_t)a.D, (cuuint64_t)G, (cuuint64_t)a.N, (cuuint64_t)a.H_kv, (cuuint64_t)a.B};
  cuuint64_t strides[4] = {G > 1 ? (cuuint64_t)a.q_strides[1] * es : any, a.N > 1 ? (cuuint64_t)a.q_strides[2] * es : any,
                           a.H_kv > 1 ? (cuuint64_t)a.q_strides[1] * es * (cuuint64_t)G : any, a.B > 1 ? (cuuint64_t)a.q_strides[0] * es : any};
  cuuint32_t box[5] = {64, (cuuint32_t)G, (cuuint32_t)tokens, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(m, a.dtype == CHILL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(a.q), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return CHILL_OK;
  snprintf(g_cuda_err, sizeof(g_cuda_err), "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return CHILL_E_CUDA;
}

// Rows can be moved in 16-byte vectors.
static bool wide(const void* p, const int64_t* st, size_t es) {
  if (st[3] != 1 || reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int d = 0; d < 3; ++d)
    if ((st[d] * (int64_t)es) % 16 != 0) return false;
  return true;
}

template <class M>
static int launch_typed(int dtype, int kernel, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st) {
  if (dtype == CHILL_F32) return launch_cached<M, CHILL_F32>(kernel, p, maps, grid, cum, st);
  if (dtype == CHILL_F16) return launch_cached<M, CHILL_F16>(kernel, p, maps, grid, cum, st);
  return launch_cached<M, CHILL_BF16>(kernel, p, maps, grid, cum, st);
}

static int cached_fwd(const chill_cached_args& a, cudaStream_t st) {
  Plan c;
  int rc = make_plan(a, c);
  if (rc != CHILL_OK) return rc;
  if (a.workspace == nullptr || a.workspace_bytes < c.bytes || reinterpret_cast<uintptr_t>(a.workspace) % 256 != 0) return CHILL_E_INVALID;
  const size_t es = esize(a.dtype);
  CachedP p{};
  p.B = a.B; p.H = a.H; p.Hkv = a.H_kv; p.G = a.H / a.H_kv; p.N = a.N; p.D = a.D;
  p.page = a.page_size; p.num_pages = a.num_pages; p.width = a.table_width; p.box = box_rows(a.page_size);
  p.wide_kv = wide(a.k_cache, a.k_cache_strides, es) && wide(a.v_cache, a.v_cache_strides, es);
  p.wide_q = wide(a.q, a.q_strides, es); p.wide_o = wide(a.o, a.o_strides, es);
  p.rows = c.rows; p.row_tiles = c.row_tiles; p.words = (a.N + 31) / 32;
  p.whole = c.whole; p.pad = c.pad; p.min_share = c.min_share; p.tail_shares = c.tail_shares;
  p.scale_log2 = a.sm_scale * kLog2e;
  p.margs = to_mask_args(a.mask, (long long)kMaxLen);
  p.q = to_ref(a.q, a.q_strides); p.k = to_ref(a.k_cache, a.k_cache_strides); p.v = to_ref(a.v_cache, a.v_cache_strides);
  p.o = to_ref(a.o, a.o_strides);
  p.lse = a.lse; p.lse_sb = a.lse_strides[0]; p.lse_sh = a.lse_strides[1]; p.lse_sl = a.lse_strides[2];
  p.table = a.table; p.table_sb = a.table_stride; p.lens = a.lens; p.new_lens = a.new_lens;
  p.positions = a.positions; p.ancestors = a.ancestors;
  char* w = (char*)a.workspace;
  int* cum = c.scan ? (int*)(w + c.cum) : nullptr;
  p.cum = cum;
  p.queue = (int*)(w + c.queue); p.seams = (Seam*)(w + c.seams); p.part_ml = (float2*)(w + c.ml); p.part_o = (float*)(w + c.o);
  p.status = device_status_ptr();
  if (p.status == nullptr) return cuda_fail(cudaGetLastError(), "status symbol");
  CUtensorMap maps[3];
  if (c.kernel != CHILL_CACHED_CUDA_CORES) {
    if ((rc = make_map(&maps[0], a.k_cache, a.k_cache_strides, a.num_pages, a.H_kv, a.page_size, a.D, a.dtype, p.box)) != CHILL_OK) return rc;
    if ((rc = make_map(&maps[1], a.v_cache, a.v_cache_strides, a.num_pages, a.H_kv, a.page_size, a.D, a.dtype, p.box)) != CHILL_OK) return rc;
  }
  if (c.kernel == CHILL_CACHED_TILES && (rc = make_q_map(&maps[2], a, tile_rows(p.G) / p.G)) != CHILL_OK) return rc;
  int e = 0;
  CHILL_MASK_SWITCH(a.mask.id, (e = launch_typed<MaskT>(a.dtype, c.kernel, p, maps, c.grid, cum, st)))
  if (e == 0) count_launches(1 + (c.scan || c.tail_shares > 0) + (c.grid > 1 && !c.whole));
  return e == 0 ? CHILL_OK : cuda_fail((cudaError_t)e, "cached attention launch");
}

}  // namespace cache
}  // namespace chill

using namespace chill;

extern "C" {

size_t chill_cached_workspace_bytes(const chill_cached_args* a) {
  cache::Plan c;
  return cache::check_cached(a, false) == CHILL_OK && cache::make_plan(*a, c) == CHILL_OK ? c.bytes : 0;
}

int chill_cached_kernel(const chill_cached_args* a) {
  const int st = cache::check_cached(a, true);
  return st != CHILL_OK ? st : cache::cached_kernel(*a);
}

int chill_cached_fwd(const chill_cached_args* a, void* stream) {
  const int st = cache::check_cached(a, true);
  return st != CHILL_OK ? st : cache::cached_fwd(*a, (cudaStream_t)stream);
}

int chill_cache_read_device_status(void) {
  int* p = device_status_ptr();
  if (p == nullptr) return CHILL_E_CUDA;
  int v = 0;
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) return cuda_fail(e, "synchronize");
  e = cudaMemcpy(&v, p, sizeof(int), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return cuda_fail(e, "status read");
  if (v != 0) {
    const int zero = 0;
    cudaMemcpy(p, &zero, sizeof(int), cudaMemcpyHostToDevice);
  }
  return v;
}

unsigned long long chill_cache_launch_count(void) { return g_launches.load(); }
const char* chill_cache_last_cuda_error(void) { return g_cuda_err; }
int chill_cache_abi_version(void) { return CHILL_CACHE_ABI_VERSION; }

}  // extern "C"
