// What the C entry points of a kernel library share: error and launch records, checks, conversions, TMA descriptors, the switch over
// the mask functors.  Included once by the file that defines a library's entry points (chill_abi.cu, cache_abi.cu): the records are
// each library's own.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdio.h>
#include <string.h>

#include <atomic>

#include "chill_b200.h"
#include "generic.cuh"

namespace chill {

static thread_local char g_cuda_err[256] = "";
__device__ int g_device_status = 0;
static std::atomic<unsigned long long> g_launches{0};  // kernels launched by this library (chill_launch_count)

static int cuda_fail(cudaError_t e, const char* what) {
  snprintf(g_cuda_err, sizeof(g_cuda_err), "%s: %s", what, cudaGetErrorString(e));
  return CHILL_E_CUDA;
}

static int* device_status_ptr() {
  // one word per device (the symbol is instantiated in every device's module image), asked for each time (33 ns): an address that is kept is
  // a stale one after a reset of the device
  int* p = nullptr;
  if (cudaGetSymbolAddress((void**)&p, g_device_status) != cudaSuccess) return nullptr;
  return p;
}

static size_t esize(int dtype) { return dtype == CHILL_F32 ? 4 : 2; }

static int check_mask(const chill_mask_desc& m) {
  if (m.n_args < 0 || m.n_args > CHILL_MAX_MASK_ARGS) return CHILL_E_INVALID;
#ifdef CHILL_CUSTOM_MASK
  if (m.id < 0 || m.id > CHILL_MASK_CUSTOM) return CHILL_E_UNSUPPORTED;
#else
  if (m.id < 0 || m.id >= CHILL_MASK_CUSTOM) return CHILL_E_UNSUPPORTED;
#endif
  if (m.id == CHILL_MASK_CHUNKWISE && (m.n_args < 2 || m.i[0] <= 0)) return CHILL_E_INVALID;
  if (m.id == CHILL_MASK_SLIDING && m.n_args < 2) return CHILL_E_INVALID;
  if (m.id == CHILL_MASK_PREFIXLM && m.n_args < 1) return CHILL_E_INVALID;
  return CHILL_OK;
}

// The functors do their index arithmetic in 32 bits (position + constant), so the 64-bit constants of the ABI are
// saturated first.  For the built-in masks every constant is a distance or a size measured in positions, and any value
// beyond +-seq_len selects the same pairs as +-seq_len itself, so they are clamped there ("unbounded" written as
// 2**31 - 1 or 2**40 stays unbounded).  Constants of a custom functor are saturated to +-2^30, which still leaves
// room for adding a position.
static MaskArgs to_mask_args(const chill_mask_desc& m, long long seq_len) {
  MaskArgs a;
  const long long lim = (m.id >= 0 && m.id < CHILL_MASK_CUSTOM && seq_len > 0) ? seq_len : (1ll << 30);
  for (int i = 0; i < 8; ++i) {
    long long v = i < m.n_args ? (long long)m.i[i] : 0;
    v = v > lim ? lim : (v < -lim ? -lim : v);
    a.i[i] = (int)v;
    a.f[i] = i < m.n_args ? (float)m.f[i] : 0.f;
  }
  if (m.id == CHILL_MASK_CHUNKWISE && a.i[0] > 0 && seq_len > 0) {
    // back_contexts counts chunks: more chunks than the sequence has changes nothing, and (chunk + back + 1) * size
    // then stays far below 2^31
    const int n_chunks = (int)((seq_len + a.i[0] - 1) / a.i[0]);
    a.i[1] = a.i[1] > n_chunks ? n_chunks : (a.i[1] < -n_chunks ? -n_chunks : a.i[1]);
  }
  return a;
}

static TRef to_ref(const void* p, const int64_t* st) {
  TRef r;
  r.p = const_cast<void*>(p);
  r.sb = st[0]; r.sh = st[1]; r.sl = st[2]; r.sd = st[3];
  return r;
}

// A [B][H][L][D] tensor can be described to TMA when channels are contiguous and everything
// else is 16-byte aligned.
static bool tma_ok(const void* p, const int64_t* st, int B, int H, int L, size_t es) {
  if (st[3] != 1) return false;
  if (((uintptr_t)p) % 16 != 0) return false;
  if ((st[2] * (int64_t)es) % 16 != 0 || st[2] <= 0) return false;
  if (H > 1 && ((st[1] * (int64_t)es) % 16 != 0 || st[1] <= 0)) return false;
  if (B > 1 && ((st[0] * (int64_t)es) % 16 != 0 || st[0] <= 0)) return false;
  (void)L;
  return true;
}

// ------------------------------------------------------------------------ TMA encoding
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  }
  return fn;
}

// Box = 64 channels x `box_rows` positions of one (batch, head), 128B swizzle.
static int make_map(CUtensorMap* m, const void* p, const int64_t* st, int B, int H, int L, int D, int dtype,
                    int box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "cuTensorMapEncodeTiled entry point not available");
    return CHILL_E_CUDA;
  }
  const cuuint64_t es = esize(dtype);
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)L, (cuuint64_t)H, (cuuint64_t)B};
  const cuuint64_t row = (cuuint64_t)st[2] * es;
  cuuint64_t strides[3] = {row, H > 1 ? (cuuint64_t)st[1] * es : row * (cuuint64_t)L,
                           B > 1 ? (cuuint64_t)st[0] * es : row * (cuuint64_t)L * (cuuint64_t)H};
  cuuint32_t box[4] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows, 1, 1};  // 128-byte rows
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == CHILL_BF16   ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                 : dtype == CHILL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  CUresult r = fn(m, dt, 4, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(g_cuda_err, sizeof(g_cuda_err), "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return CHILL_E_CUDA;
  }
  return CHILL_OK;
}

// --------------------------------------------------------------------------- dispatch
#ifdef CHILL_CUSTOM_MASK
#define CHILL_CUSTOM_CASE(CALL) \
  case CHILL_MASK_CUSTOM: { using MaskT = CHILL_CUSTOM_MASK; CALL; break; }
#else
#define CHILL_CUSTOM_CASE(CALL)
#endif

#ifdef CHILL_CUSTOM_MASK_ONLY  // a library with the kernels of the custom functor alone
#define CHILL_BUILTIN_CASES(CALL)
#else
#define CHILL_BUILTIN_CASES(CALL)                                          \
    case CHILL_MASK_FULL: { using MaskT = FullMask; CALL; break; }         \
    case CHILL_MASK_CAUSAL: { using MaskT = CausalMask; CALL; break; }     \
    case CHILL_MASK_SLIDING: { using MaskT = SlidingWindowMask; CALL; break; } \
    case CHILL_MASK_CHUNKWISE: { using MaskT = ChunkwiseMask; CALL; break; } \
    case CHILL_MASK_PREFIXLM: { using MaskT = PrefixLMMask; CALL; break; }
#endif

#define CHILL_MASK_SWITCH(ID, CALL) CHILL_MASK_SWITCH_OR(ID, CALL, return CHILL_E_UNSUPPORTED)
#define CHILL_MASK_SWITCH_OR(ID, CALL, OTHERWISE)                          \
  switch (ID) {                                                            \
    CHILL_BUILTIN_CASES(CALL)                                              \
    CHILL_CUSTOM_CASE(CALL)                                                \
    default: OTHERWISE;                                                    \
  }

#define CHILL_DTYPE_SWITCH(DT, CALL)                                  \
  switch (DT) {                                                       \
    case CHILL_F32: { using ElemT = float; CALL; break; }             \
    case CHILL_F16: { using ElemT = __half; CALL; break; }            \
    case CHILL_BF16: { using ElemT = __nv_bfloat16; CALL; break; }    \
    default: return CHILL_E_UNSUPPORTED;                              \
  }

}  // namespace chill
