// Records of libchill_decode_b200.so (include/chill_decode.h); the operators are in decode_rotary.cu, decode_beams.cu and decode_pages.cu.
#include <stdio.h>

#include <atomic>

#include "decode_common.cuh"

namespace chill {
namespace decode {

static thread_local char g_cuda_err[256] = "";
static std::atomic<unsigned long long> g_launches{0};

int record_cuda_failure(cudaError_t e, const char* what) {
  snprintf(g_cuda_err, sizeof(g_cuda_err), "%s: %s", what, cudaGetErrorString(e));
  return CHILL_E_CUDA;
}

void count_launches(int n) { g_launches += n; }

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n;
}

}  // namespace decode
}  // namespace chill

extern "C" {

unsigned long long chill_decode_launch_count(void) { return chill::decode::g_launches.load(); }
const char* chill_decode_last_cuda_error(void) { return chill::decode::g_cuda_err; }
int chill_decode_abi_version(void) { return CHILL_DECODE_ABI_VERSION; }

}  // extern "C"
