// Host-side launchers of the attention kernels over a paged cache; each mask functor's are compiled in a translation unit of
// their own (cache_inst.cu with -DCHILL_INST_MASK=<functor>), which defines the explicit specialisations declared here.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace chill {
namespace cache {
struct CachedP;

// `kernel`: CHILL_CACHED_*.  `grid` CTAs share the work; returns a cudaError_t cast to int and adds to `launches`.
template <class M>
int launch_cached(int kernel, int dtype, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st, int* launches);

}  // namespace cache
}  // namespace chill
