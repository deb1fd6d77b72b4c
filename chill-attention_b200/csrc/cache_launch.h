// Host-side launchers of the attention kernels over a paged cache; those of one mask functor and one data type are compiled in a
// translation unit of their own (cache_inst.cu with -DCHILL_INST_MASK=<functor> -DCHILL_INST_PART=<CHILL_F32 ..>), which defines the
// explicit specialisation declared here.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace chill {
namespace cache {
struct CachedP;

// `kernel`: CHILL_CACHED_*; `grid` CTAs share the work; maps: K, V, Q; `cum`: where the prefix sums go when they have a
// launch of their own, or null.  Returns a cudaError_t cast to int.
template <class M, int DTYPE>
int launch_cached(int kernel, const CachedP& p, const CUtensorMap* maps, int grid, int* cum, cudaStream_t st);

}  // namespace cache
}  // namespace chill
