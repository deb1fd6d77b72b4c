// Instantiates the attention kernels over a paged cache for ONE mask functor and ONE data type: compile with
//   -DCHILL_INST_MASK=<functor struct> -DCHILL_INST_PART=<CHILL_F32, CHILL_F16 or CHILL_BF16, as a number>
#include "cache_launch.h"
#include "cache_rows.cuh"
#include "cache_simt.cuh"
#include "cache_tiles.cuh"
#include "chill_cache.h"
#include "tc_launch.h"

#if !defined(CHILL_INST_MASK) || !defined(CHILL_INST_PART)
#error "define CHILL_INST_MASK and CHILL_INST_PART"
#endif

namespace chill {
namespace cache {

using InstMask = CHILL_INST_MASK;
using InstType = std::conditional_t<CHILL_INST_PART == CHILL_F32, float, std::conditional_t<CHILL_INST_PART == CHILL_F16, __half, __nv_bfloat16>>;

template <typename T, int DP>
static int launch_simt(const CachedP& p, int grid, cudaStream_t st) {
  auto kern = cached_simt_kernel<T, DP, InstMask>;
  constexpr int smem = SimtSmem<DP>::kBytes;
  static_assert(smem <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, smem, /*prefer_max_carveout=*/true);
  if (e != cudaSuccess) return (int)e;
  kern<<<grid, kSimtThreads, smem, st>>>(p);
  return (int)cudaGetLastError();
}

template <typename T, int DP, int MT>
static int launch_rows(const CachedP& p, const CUtensorMap* maps, int grid, cudaStream_t st) {
  auto kern = cached_rows_kernel<T, DP, MT, InstMask>;
  constexpr int smem = RowsShape<DP, MT>::kDynamic;
  static_assert(smem <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, smem, /*prefer_max_carveout=*/true);
  if (e != cudaSuccess) return (int)e;
  kern<<<grid, kRowsThreads, smem, st>>>(maps[0], maps[1], p);
  return (int)cudaGetLastError();
}

template <typename T, int DP>
static int launch_tiles(const CachedP& p, const CUtensorMap* maps, int grid, cudaStream_t st) {
  auto kern = cached_tiles_kernel<T, DP, InstMask>;
  constexpr int smem = TilesShape<DP>::kDynamic;
  static_assert(smem <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, smem, /*prefer_max_carveout=*/true);
  if (e != cudaSuccess) return (int)e;
  kern<<<grid, kTilesThreads, smem, st>>>(maps[0], maps[1], p);
  return (int)cudaGetLastError();
}

template <typename T>
static int launch_typed(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (kernel == CHILL_CACHED_TILES) {
      if (p.D > 128) return launch_tiles<T, 256>(p, maps, grid, st);
      return p.D > 64 ? launch_tiles<T, 128>(p, maps, grid, st) : launch_tiles<T, 64>(p, maps, grid, st);
    }
    if (kernel == CHILL_CACHED_ROWS) {
      if (p.D > 128) return launch_rows<T, 256, 1>(p, maps, grid, st);
      if (p.D > 64) return p.rows == 16 ? launch_rows<T, 128, 1>(p, maps, grid, st) : launch_rows<T, 128, 2>(p, maps, grid, st);
      return p.rows == 16 ? launch_rows<T, 64, 1>(p, maps, grid, st) : launch_rows<T, 64, 2>(p, maps, grid, st);
    }
  }
  if (kernel != CHILL_CACHED_CUDA_CORES) return (int)cudaErrorInvalidValue;
  if (p.D <= 32) return launch_simt<T, 32>(p, grid, st);
  if (p.D <= 64) return launch_simt<T, 64>(p, grid, st);
  if (p.D <= 128) return launch_simt<T, 128>(p, grid, st);
  return launch_simt<T, 256>(p, grid, st);
}

// The parts are joined by a kernel whose launch overlaps the end of the first one; it waits for that before it reads.
template <typename T>
static int launch_join(const CachedP& p, int grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)imax(grid - 1, 1), (unsigned)(p.rows / 16));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, join_kernel<T>, p, grid);
}

template <>
int launch_cached<InstMask, CHILL_INST_PART>(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st, int* launches) {
  if (cum != nullptr) {
    scan_kernel<InstMask><<<1, 1024, 0, st>>>(p, cum);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    *launches += 1;
  }
  int e = launch_typed<InstType>(kernel, p, maps, grid, st);
  if (e != 0) return e;
  *launches += 1;
  if (grid == 1) return 0;  // nothing is cut
  e = launch_join<InstType>(p, grid, st);
  if (e == 0) *launches += 1;
  return e;
}

}  // namespace cache
}  // namespace chill
