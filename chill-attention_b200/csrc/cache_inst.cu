// Instantiates the attention kernels over a paged cache for ONE mask functor: compile with -DCHILL_INST_MASK=<functor struct>
#include "cache_launch.h"
#include "cache_simt.cuh"
#include "chill_b200.h"
#include "tc_launch.h"

#ifndef CHILL_INST_MASK
#error "define CHILL_INST_MASK"
#endif

namespace chill {
namespace cache {

using InstMask = CHILL_INST_MASK;

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

template <typename T>
static int launch_typed(int kernel, const CachedP& p, const CUtensorMap*, int grid, cudaStream_t st) {
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

template <typename T>
static int launch_all(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, cudaStream_t st, int* launches) {
  int e = launch_typed<T>(kernel, p, maps, grid, st);
  if (e != 0) return e;
  *launches += 1;
  if (grid == 1) return 0;  // nothing is cut
  e = launch_join<T>(p, grid, st);
  if (e == 0) *launches += 1;
  return e;
}

template <>
int launch_cached<InstMask>(int kernel, int dtype, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st, int* launches) {
  if (cum != nullptr) {
    scan_kernel<InstMask><<<1, 1024, 0, st>>>(p, cum);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    *launches += 1;
  }
  if (dtype == CHILL_F32) return launch_all<float>(kernel, p, maps, grid, st, launches);
  if (dtype == CHILL_F16) return launch_all<__half>(kernel, p, maps, grid, st, launches);
  return launch_all<__nv_bfloat16>(kernel, p, maps, grid, st, launches);
}

}  // namespace cache
}  // namespace chill
