// Attention over a paged cache: checks of the arguments, choice of the kernel, workspace, launch.  Included by chill_abi.cu, whose
// helpers it uses.
#pragma once

static int check_cached(const chill_cached_args* a, bool pointers) {
  if (a == nullptr || a->B <= 0 || a->H <= 0 || a->H_kv <= 0 || a->N <= 0 || a->D <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->table_width <= 0)
    return CHILL_E_INVALID;
  if (a->H % a->H_kv != 0) return CHILL_E_INVALID;
  if (a->dtype != CHILL_F32 && a->dtype != CHILL_F16 && a->dtype != CHILL_BF16) return CHILL_E_UNSUPPORTED;
  if (a->D > kMaxD || a->D % 16 != 0) return CHILL_E_UNSUPPORTED;
  if (a->B > 65535 || a->H > 65535 || a->N > cache::kMaxLen / 2 || (long long)a->N * (a->H / a->H_kv) > cache::kMaxLen ||
      (long long)a->num_pages * a->page_size > 0x7fffffffll || (long long)a->table_width * a->page_size > cache::kMaxLen)
    return CHILL_E_TOO_LARGE;
  if (!(a->sm_scale > 0.f) || a->sm_scale > 3e38f) return CHILL_E_INVALID;
  const int st = check_mask(a->mask);
  if (st != CHILL_OK) return st;
  if (!pointers) return CHILL_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->o || !a->table || !a->lens || !a->new_lens) return CHILL_E_INVALID;
  if (a->ancestors != nullptr && a->positions == nullptr) return CHILL_E_INVALID;
  return CHILL_OK;
}

// Kernel, tiles, CTAs and workspace of a call: from the sizes that the host knows.
struct CachedPlan {
  int kernel, rows, row_tiles, grid, min_share;
  bool scan;  // prefix sums by a launch of their own
  size_t seam, all, cum, ml, o, bytes;
};

static int cached_kernel(const chill_cached_args&) { return CHILL_CACHED_CUDA_CORES; }

static int plan_cached(const chill_cached_args& a, CachedPlan& c) {
  c.kernel = cached_kernel(a);
  c.rows = 16;
  c.min_share = 2;
  c.grid = sm_count() * (a.D <= 64 ? 4 : (a.D <= 128 ? 2 : 1));
  c.row_tiles = (int)(((long long)a.N * (a.H / a.H_kv) + c.rows - 1) / c.rows);
  const long long entries = (long long)a.B * c.row_tiles;
  const long long keys = imin(a.table_width * a.page_size, cache::kMaxLen);
  if (entries * a.H_kv * (keys / cache::kKeyTile + 2) > 0x7fffffffll) return CHILL_E_TOO_LARGE;
  c.scan = entries > cache::kScanEntries;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  c.seam = 0;
  c.all = up((size_t)c.grid * sizeof(int4));
  c.cum = c.all + 256;
  c.ml = c.cum + (c.scan ? up((size_t)(entries + 1) * 4) : 0);
  c.o = c.ml + up((size_t)2 * c.grid * c.rows * sizeof(float2));
  c.bytes = c.o + up((size_t)2 * c.grid * c.rows * a.D * sizeof(float));
  return CHILL_OK;
}

static int cached_fwd(const chill_cached_args& a, cudaStream_t st) {
  CachedPlan c;
  int rc = plan_cached(a, c);
  if (rc != CHILL_OK) return rc;
  if (a.workspace == nullptr || a.workspace_bytes < c.bytes || reinterpret_cast<uintptr_t>(a.workspace) % 256 != 0) return CHILL_E_INVALID;
  cache::CachedP p{};
  p.B = a.B; p.H = a.H; p.Hkv = a.H_kv; p.G = a.H / a.H_kv; p.N = a.N; p.D = a.D;
  p.page = a.page_size; p.num_pages = a.num_pages; p.width = a.table_width;
  p.rows = c.rows; p.row_tiles = c.row_tiles; p.words = (a.N + 31) / 32; p.min_share = c.min_share;
  p.scale_log2 = a.sm_scale * kLog2e;
  p.margs = to_mask_args(a.mask, (long long)cache::kMaxLen);
  p.q = to_ref(a.q, a.q_strides); p.k = to_ref(a.k_cache, a.k_cache_strides); p.v = to_ref(a.v_cache, a.v_cache_strides);
  p.o = to_ref(a.o, a.o_strides);
  p.lse = a.lse; p.lse_sb = a.lse_strides[0]; p.lse_sh = a.lse_strides[1]; p.lse_sl = a.lse_strides[2];
  p.table = a.table; p.table_sb = a.table_stride; p.lens = a.lens; p.new_lens = a.new_lens;
  p.positions = a.positions; p.ancestors = a.ancestors;
  char* w = (char*)a.workspace;
  p.cum = c.scan ? (const int*)(w + c.cum) : nullptr;
  p.seam = (int4*)(w + c.seam); p.all = (int*)(w + c.all); p.part_ml = (float2*)(w + c.ml); p.part_o = (float*)(w + c.o);
  p.status = device_status_ptr();
  if (p.status == nullptr) return cuda_fail(cudaGetLastError(), "status symbol");
  int e = 0, launches = 0;
  CHILL_MASK_SWITCH(a.mask.id, (e = cache::launch_cached<MaskT>(c.kernel, a.dtype, p, nullptr, c.grid, c.scan ? (int*)(w + c.cum) : nullptr, st, &launches)))
  g_launches += launches;
  return e == 0 ? CHILL_OK : cuda_fail((cudaError_t)e, "cached attention launch");
}
