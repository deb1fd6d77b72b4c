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
  if (!(a->sm_scale > 0.f) || a->sm_scale > 3e38f) return CHILL_E_INVALID;
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

// CHILL_CACHED_*: few rows go through mma.sync, which reads the keys once for all of them, many through tiles of 128 rows.
static int cached_kernel(const chill_cached_args& a) {
  if (a.dtype == CHILL_F32 || (a.flags & CHILL_FLAG_FORCE_GENERIC) || box_rows(a.page_size) == 0) return CHILL_CACHED_CUDA_CORES;
  const size_t es = esize(a.dtype);
  if (!tma_ok(a.k_cache, a.k_cache_strides, a.num_pages, a.H_kv, a.page_size, es) || !tma_ok(a.v_cache, a.v_cache_strides, a.num_pages, a.H_kv, a.page_size, es))
    return CHILL_CACHED_CUDA_CORES;
  return (long long)a.N * (a.H / a.H_kv) <= (a.D <= 128 ? 32 : 16) ? CHILL_CACHED_ROWS : CHILL_CACHED_TILES;
}

// Kernel, tiles, CTAs and workspace of a call, from the sizes that the host knows.
struct Plan {
  int kernel, rows, row_tiles, grid, min_share;
  bool scan;  // prefix sums by a launch of their own
  size_t seam, all, cum, ml, o, bytes;
};

static int make_plan(const chill_cached_args& a, Plan& c) {
  const long long group_rows = (long long)a.N * (a.H / a.H_kv);
  c.kernel = cached_kernel(a);
  c.min_share = 2;
  if (c.kernel == CHILL_CACHED_CUDA_CORES) {
    c.rows = 16;
    c.grid = sm_count() * (a.D <= 64 ? 4 : (a.D <= 128 ? 2 : 1));
  } else {
    c.rows = c.kernel == CHILL_CACHED_TILES ? 128 : (group_rows <= 16 ? 16 : 32);
    c.grid = sm_count() * (a.D <= 128 ? 2 : 1);
  }
  c.row_tiles = (int)((group_rows + c.rows - 1) / c.rows);
  const long long entries = (long long)a.B * c.row_tiles;
  const long long keys = (long long)a.table_width * a.page_size;
  if (entries * a.H_kv * (keys / kKeyTile + 2) > 0x7fffffffll) return CHILL_E_TOO_LARGE;
  c.scan = entries > kScanEntries;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  c.seam = 0;
  c.all = up((size_t)c.grid * sizeof(int4));
  c.cum = c.all + 256;
  c.ml = c.cum + (c.scan ? up((size_t)(entries + 1) * 4) : 0);
  c.o = c.ml + up((size_t)2 * c.grid * c.rows * sizeof(float2));
  c.bytes = c.o + up((size_t)2 * c.grid * c.rows * a.D * sizeof(float));
  return CHILL_OK;
}

// Rows can be moved in 16-byte vectors.
static bool wide(const void* p, const int64_t* st, size_t es) {
  if (st[3] != 1 || reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  for (int d = 0; d < 3; ++d)
    if ((st[d] * (int64_t)es) % 16 != 0) return false;
  return true;
}

template <class M>
static int launch_typed(int dtype, int kernel, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st, int* launches) {
  if (dtype == CHILL_F32) return launch_cached<M, CHILL_F32>(kernel, p, maps, grid, cum, st, launches);
  if (dtype == CHILL_F16) return launch_cached<M, CHILL_F16>(kernel, p, maps, grid, cum, st, launches);
  return launch_cached<M, CHILL_BF16>(kernel, p, maps, grid, cum, st, launches);
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
  p.wide_q = wide(a.q, a.q_strides, es); p.wide_o = wide(a.o, a.o_strides, es);
  p.rows = c.rows; p.row_tiles = c.row_tiles; p.words = (a.N + 31) / 32; p.min_share = c.min_share;
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
  p.seam = (int4*)(w + c.seam); p.all = (int*)(w + c.all); p.part_ml = (float2*)(w + c.ml); p.part_o = (float*)(w + c.o);
  p.status = device_status_ptr();
  if (p.status == nullptr) return cuda_fail(cudaGetLastError(), "status symbol");
  CUtensorMap maps[2];
  if (c.kernel != CHILL_CACHED_CUDA_CORES) {
    if ((rc = make_map(&maps[0], a.k_cache, a.k_cache_strides, a.num_pages, a.H_kv, a.page_size, a.D, a.dtype, p.box)) != CHILL_OK) return rc;
    if ((rc = make_map(&maps[1], a.v_cache, a.v_cache_strides, a.num_pages, a.H_kv, a.page_size, a.D, a.dtype, p.box)) != CHILL_OK) return rc;
  }
  int e = 0, launches = 0;
  CHILL_MASK_SWITCH(a.mask.id, (e = launch_typed<MaskT>(a.dtype, c.kernel, p, maps, c.grid, cum, st, &launches)))
  count_launches(launches);
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
