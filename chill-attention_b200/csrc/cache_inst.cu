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

// `behind`: launched while the kernel before it in the stream, one of this call, runs; it waits for that where it needs its results.
// The first kernel of a call never is: what runs before it is not known.
template <class... Args, class... Given>
static int launch(bool behind, void (*kern)(Args...), dim3 grid, int threads, int smem, cudaStream_t st, const Given&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = behind ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kern, Args(args)...);
}

template <typename T, int DP, int RT>
static int launch_simt_many(const CachedP& p, int grid, bool behind, cudaStream_t st) {
  auto kern = cached_simt_many_kernel<T, DP, RT, InstMask>;
  constexpr int smem = SimtSmem<DP, RT>::kBytes;
  static_assert(smem <= 232448 && SimtSmem<DP, RT>::kCtasPerSm * (smem + 1024) <= 233472, "shared memory of an SM");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, smem, /*prefer_max_carveout=*/true);
  return e != cudaSuccess ? (int)e : launch(behind, kern, dim3((unsigned)grid), kSimtThreads, smem, st, p);
}

template <typename T, int DP>
static int launch_simt(const CachedP& p, int grid, bool behind, cudaStream_t st) {
  const dim3 blocks((unsigned)grid);
  if (p.rows == 2 && p.whole) return launch(behind, cached_simt_few_kernel<T, DP, 2, 8, InstMask>, blocks, 256, 0, st, p);
  if (p.rows == 2) return launch(behind, cached_simt_few_kernel<T, DP, 2, 4, InstMask>, blocks, 128, 0, st, p);
  if (p.rows == 4 && p.whole) return launch(behind, cached_simt_few_kernel<T, DP, 4, 8, InstMask>, blocks, 256, 0, st, p);
  if (p.rows == 4) return launch(behind, cached_simt_few_kernel<T, DP, 4, 4, InstMask>, blocks, 128, 0, st, p);
  if (p.rows == 8) return launch_simt_many<T, DP, 1>(p, grid, behind, st);
  return p.rows == 16 ? launch_simt_many<T, DP, 2>(p, grid, behind, st) : launch_simt_many<T, DP, 4>(p, grid, behind, st);
}

template <typename T, int DP, int MT>
static int launch_rows(const CachedP& p, const CUtensorMap* maps, int grid, bool behind, cudaStream_t st) {
  auto kern = cached_rows_kernel<T, DP, MT, InstMask>;
  constexpr int smem = RowsShape<DP, MT>::kDynamic;
  static_assert(smem <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, smem, /*prefer_max_carveout=*/true);
  return e != cudaSuccess ? (int)e : launch(behind, kern, dim3((unsigned)grid), kRowsThreads, smem, st, maps[0], maps[1], p);
}

template <typename T, int DP, int NQ>
static int launch_tiles(const CachedP& p, const CUtensorMap* maps, int grid, bool behind, cudaStream_t st) {
  using S = TilesShape<DP, NQ>;
  auto kern = cached_tiles_kernel<T, DP, NQ, InstMask>;
  static_assert(S::kDynamic <= 232448, "exceeds the 227 KB of shared memory a CTA can opt in to");
  struct Tag {};
  cudaError_t e = ensure_dynamic_smem<Tag>(kern, S::kDynamic, /*prefer_max_carveout=*/true);
  if (e != cudaSuccess) return (int)e;
  return launch(behind, kern, dim3((unsigned)grid), S::kThreads, S::kDynamic, st, maps[2], maps[0], maps[1], p);
}

template <typename T>
static int launch_typed(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, bool behind, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (kernel == CHILL_CACHED_TILES) {
      const bool two = p.rows > kTileRows;
      if (p.D > 128) return launch_tiles<T, 256, 1>(p, maps, grid, behind, st);
      if (p.D > 64) return two ? launch_tiles<T, 128, 2>(p, maps, grid, behind, st) : launch_tiles<T, 128, 1>(p, maps, grid, behind, st);
      return two ? launch_tiles<T, 64, 2>(p, maps, grid, behind, st) : launch_tiles<T, 64, 1>(p, maps, grid, behind, st);
    }
    if (kernel == CHILL_CACHED_ROWS) {
      if (p.D > 128) return launch_rows<T, 256, 1>(p, maps, grid, behind, st);
      if (p.D > 64) return p.rows == 16 ? launch_rows<T, 128, 1>(p, maps, grid, behind, st) : launch_rows<T, 128, 2>(p, maps, grid, behind, st);
      return p.rows == 16 ? launch_rows<T, 64, 1>(p, maps, grid, behind, st) : launch_rows<T, 64, 2>(p, maps, grid, behind, st);
    }
  }
  if (kernel != CHILL_CACHED_CUDA_CORES) return (int)cudaErrorInvalidValue;
  if (p.D <= 32) return launch_simt<T, 32>(p, grid, behind, st);
  if (p.D <= 64) return launch_simt<T, 64>(p, grid, behind, st);
  if (p.D <= 128) return launch_simt<T, 128>(p, grid, behind, st);
  return launch_simt<T, 256>(p, grid, behind, st);
}

template <>
int launch_cached<InstMask, CHILL_INST_PART>(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st) {
  const bool prepare = cum != nullptr || p.tail_shares > 0;
  if (prepare) {
    prepare_kernel<InstMask><<<1, cum != nullptr ? kScanThreads : 32, 0, st>>>(p, cum);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
  }
  const int e = launch_typed<InstType>(kernel, p, maps, grid, prepare, st);
  if (e != 0 || grid == 1 || p.whole) return e;  // nothing is cut
  const int shares = grid + p.tail_shares;
  if (kernel == CHILL_CACHED_TILES) return launch(true, join_many_kernel<InstType>, dim3((unsigned)shares, (unsigned)((p.rows + 31) / 32)), kJoinThreads, 0, st, p);
  // units that are far fewer than shares have many parts each
  const long long rows = imin(p.rows, p.N * p.G), units = (long long)p.B * p.row_tiles * p.Hkv;
  const int many = 4 * units < shares;
  const dim3 blocks((unsigned)imin(shares, (many ? 1 : 3) * sm_count()), (unsigned)(many ? rows : (rows + 7) / 8));
  if (p.D > 128) return launch(true, join_few_kernel<InstType, 2>, blocks, kJoinThreads, 0, st, p, many, shares);
  return launch(true, join_few_kernel<InstType, 1>, blocks, kJoinThreads, 0, st, p, many, shares);
}

}  // namespace cache
}  // namespace chill
