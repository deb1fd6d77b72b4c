// What the sources of libchill_decode_b200.so share (include/chill_decode.h).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "chill_decode.h"

namespace chill {
namespace decode {

int record_cuda_failure(cudaError_t e, const char* what);  // decode_abi.cu
void count_launches(int n);                                // decode_abi.cu
int sm_count();                                            // decode_abi.cu: of the current device

constexpr int kMaxLen = 1 << 29;  // positions; three of them added stay below 2^31
constexpr int kMaxRequests = 65535;

__host__ __device__ __forceinline__ int imin(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int imax(int a, int b) { return a > b ? a : b; }
__device__ __forceinline__ int clamp_len(int x) { return imin(imax(x, 0), kMaxLen); }

template <class T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};

// V elements that are moved in one access.
template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
  T x[V];
};

// Of what nobody reads again in the same kernel: 16 bytes past the caches' usual order.  With plain loads and stores 20 % longer (rotation of q and k of (8, 16, 4096, 128) in bf16).
template <class V>
__device__ __forceinline__ V load_once(const char* p) {
  if constexpr (sizeof(V) == 16) {
    const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(p));
    return *reinterpret_cast<const V*>(&raw);
  } else {
    return *reinterpret_cast<const V*>(p);
  }
}
template <class V>
__device__ __forceinline__ void store_once(char* p, const V& v) {
  if constexpr (sizeof(V) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
  else *reinterpret_cast<V*>(p) = v;
}

inline int elem_size(int dtype) { return dtype == CHILL_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == CHILL_F32 || dtype == CHILL_F16 || dtype == CHILL_BF16; }

// The largest vector (bytes, up to 16) in which the rows of a tensor can be moved: channels adjacent, base and strides multiples of it.
inline int row_vector(const void* p, const int64_t* strides, int outer, int es) {
  if (strides[outer] != 1) return es;
  for (int bytes = 16; bytes > es; bytes /= 2) {
    bool fits = reinterpret_cast<uintptr_t>(p) % bytes == 0;
    for (int d = 0; d < outer; ++d) fits = fits && (strides[d] * es) % bytes == 0;
    if (fits) return bytes;
  }
  return es;
}

}  // namespace decode
}  // namespace chill
