// Rotary positions: q and k turned by the angles of their positions, out of place (chill_rotate; with the opposite angle its backward) or k into its
// slots of a paged cache together with v (chill_rotate_append).  include/chill_decode.h has the formula.
//
// A copy with little arithmetic: every row is read and written once, so the bound is memory.  A thread owns one vector of pairs of one token and
// goes over heads with it.  The sines and cosines are the same for all heads: a block's warps, which have the same vectors of different heads, share them.  q and k of (8, 16, 4096, 128) in bf16:
// 84 us (6.4 TB/s, 0.97 of a copy's rate; 87 us where every thread works out its own); (3, 32 and 8, 5003, 128) in fp16, 96 channels turned by three axes: 52 us (0.91).  Into pages of 16, 24
// and 8 heads of 128 in fp16: 3 prompts of 5000 tokens 55 us (0.85), 4 of 1000 18.7 us (0.67; 16.5 where inputs and outputs, 81 MB, stay in L2): two waves of short CTAs, the second
// not full.  The next heads' loads ahead of this one's arithmetic, with one loop over the heads of all tensors: 178 us (pointers chosen a head, spills).
#include "decode_common.cuh"

namespace chill {
namespace decode {

constexpr int kThreads = 128;
// Vectors that a block has; its other threads have the same ones of other heads.  Narrow vectors: as many as there are threads, so that a block's accesses lie side by side
// (102 of 128 channels in halves, fp16, element by element: 31 us, with 32 vectors 50).
template <class T, int V>
constexpr int kItems = V * sizeof(T) == 16 ? 32 : kThreads;

struct RotateP {
  int B, L, H, Hkv, pairs, D, n_axes, inverse;
  int per_row;        // threads of a row: vectors of pairs, then vectors of channels that stay
  int turning;        // of these, the ones that turn
  int heads, slices;  // of q, k (and v); a warp goes over heads / slices of them
  unsigned items;     // B * L * per_row
  const float* inv_freq;
  const int *axes, *positions;
  long long pos_axis, pos_batch, pos_token;
  const char *q, *k, *v;
  char *qo, *ko, *kc, *vc;
  long long qs[4], ks[4], vs[4], qos[4], kos[4], kcs[4], vcs[4];  // bytes
  const int* slots;
  int num_pages, page;
};

// cos and sin of position * freq.  The angle in turns is formed in 64 bits and reduced there, so far positions cost no accuracy: the product of an
// integer below 2^31 and a fp32 frequency is off by at most 2^-53 of its size twice, 2^-22 turns at 2^31 radians.
__device__ __forceinline__ float2 turn(int position, float freq) {
  const double turns = (double)position * ((double)freq * 0.15915494309189533577);
  const float half = (float)(2.0 * (turns - rint(turns)));
  float2 cs;
  sincospif(half, &cs.y, &cs.x);
  return cs;
}

// kPaired: pairs (2 i, 2 i + 1); a vector of V channels is V / 2 pairs (V = 1: a thread moves a pair as two elements).  Otherwise pairs (i, i + pairs): two
// vectors.  V > 1 wants channels that lie beside each other.
template <class T, int V, bool kPaired, bool kAppend>
__global__ void __launch_bounds__(kThreads, 8) rotate_kernel(const __grid_constant__ RotateP p) {
  const unsigned at = blockIdx.x * (unsigned)kItems<T, V> + threadIdx.x % kItems<T, V>;
  const bool inside = at < p.items;
  const unsigned token = at / (unsigned)p.per_row;
  const int part = (int)(at - token * (unsigned)p.per_row);
  const int b = (int)(token / (unsigned)p.L), i = (int)(token - (unsigned)b * (unsigned)p.L);
  constexpr int kPairs = kPaired ? (V + 1) / 2 : V;  // of a thread
  constexpr bool kTwo = !kPaired || V == 1;          // two vectors of a row, `apart` channels from one another
  const bool turns = part < p.turning;
  const int first = part * kPairs;  // the thread's first pair
  const int c0 = turns ? (kPaired ? 2 * first : first) : 2 * p.pairs + (part - p.turning) * V;
  const int apart = kPaired ? 1 : p.pairs;

  // Sines and cosines, by all of the block's threads together
  constexpr int kFours = (kPairs + 1) / 2;
  __shared__ float4 both[kFours][kItems<T, V>];
  for (int i = threadIdx.x; i < kItems<T, V> * kPairs; i += kThreads) {
    const int item = i % kItems<T, V>, n = i / kItems<T, V>;
    const unsigned other = blockIdx.x * (unsigned)kItems<T, V> + (unsigned)item, its_token = other / (unsigned)p.per_row;
    const int its_part = (int)(other - its_token * (unsigned)p.per_row);
    if (other >= p.items || its_part >= p.turning) continue;
    const int pair = its_part * kPairs + n, its_b = (int)(its_token / (unsigned)p.L), its_i = (int)(its_token - (unsigned)its_b * (unsigned)p.L);
    const int axis = p.axes != nullptr ? imin(imax(p.axes[pair], 0), p.n_axes - 1) : 0;
    float2 x = turn(p.positions[axis * p.pos_axis + its_b * p.pos_batch + its_i * p.pos_token], p.inv_freq[pair]);
    if (p.inverse) x.y = -x.y;
    reinterpret_cast<float2*>(&both[n / 2][item])[n & 1] = x;
  }
  __syncthreads();
  if (!inside) return;
  float2 cs[kPairs];
#pragma unroll
  for (int n = 0; n < kPairs; n += 2) {
    const float4 x = both[n / 2][threadIdx.x % kItems<T, V>];
    cs[n] = make_float2(x.x, x.y);
    if (n + 1 < kPairs) cs[n + 1] = make_float2(x.z, x.w);
  }
  int slot = -1, page = 0, row = 0;
  if constexpr (kAppend) {
    slot = p.slots[(long long)b * p.L + i];
    if (slot >= p.num_pages * p.page) slot = -1;
    page = slot / p.page;
    row = slot - page * p.page;
  }

  const int slice = (int)blockIdx.y * (kThreads / kItems<T, V>) + (int)threadIdx.x / kItems<T, V>;
  const int h0 = (int)((long long)p.heads * slice / p.slices), h1 = (int)((long long)p.heads * (slice + 1) / p.slices);
  using VecT = Vec<T, V>;
  // Heads [from, to) of one tensor, kBatch at a time: as many loads on their way before the first store.
  auto go = [&](const char* src, long long src_head, char* dst, long long dst_head, long long src_chan, long long dst_chan, int count, bool rotate) {
    constexpr int kBatch = kTwo && V * sizeof(T) == 16 ? 2 : 4;
    for (int n0 = 0; n0 < count; n0 += kBatch) {
      VecT x[kBatch], y[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (n0 + u < count) {
          x[u] = load_once<VecT>(src + (n0 + u) * src_head);
          if (kTwo && turns) y[u] = load_once<VecT>(src + (n0 + u) * src_head + apart * src_chan);
        }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (n0 + u < count) {
          if (turns && rotate) {
#pragma unroll
            for (int n = 0; n < kPairs; ++n) {
              T* lo = kTwo ? &x[u].x[n] : &x[u].x[(2 * n) % V];
              T* hi = kTwo ? &y[u].x[n] : &x[u].x[(2 * n + 1) % V];
              const float a = Elem<T>::up(*lo), c = Elem<T>::up(*hi);
              *lo = Elem<T>::down(a * cs[n].x - c * cs[n].y);
              *hi = Elem<T>::down(c * cs[n].x + a * cs[n].y);
            }
          }
          store_once(dst + (n0 + u) * dst_head, x[u]);
          if (kTwo && turns) store_once(dst + (n0 + u) * dst_head + apart * dst_chan, y[u]);
        }
    }
  };
  if (h0 < p.H) {
    go(p.q + b * p.qs[0] + h0 * p.qs[1] + i * p.qs[2] + c0 * p.qs[3], p.qs[1], p.qo + b * p.qos[0] + h0 * p.qos[1] + i * p.qos[2] + c0 * p.qos[3],
       p.qos[1], p.qs[3], p.qos[3], imin(h1, p.H) - h0, true);
  }
  const int k0 = imax(h0 - p.H, 0), k1 = imin(h1 - p.H, p.Hkv);
  if (k0 < k1) {
    const char* src = p.k + b * p.ks[0] + k0 * p.ks[1] + i * p.ks[2] + c0 * p.ks[3];
    if constexpr (kAppend) {
      if (slot >= 0)
        go(src, p.ks[1], p.kc + page * p.kcs[0] + k0 * p.kcs[1] + row * p.kcs[2] + c0 * p.kcs[3], p.kcs[1], p.ks[3], p.kcs[3], k1 - k0, true);
    } else {
      go(src, p.ks[1], p.ko + b * p.kos[0] + k0 * p.kos[1] + i * p.kos[2] + c0 * p.kos[3], p.kos[1], p.ks[3], p.kos[3], k1 - k0, true);
    }
  }
  if constexpr (kAppend) {
    const int v0 = imax(h0 - p.H - p.Hkv, 0), v1 = h1 - p.H - p.Hkv;
    if (v0 < v1 && slot >= 0)
      go(p.v + b * p.vs[0] + v0 * p.vs[1] + i * p.vs[2] + c0 * p.vs[3], p.vs[1], p.vc + page * p.vcs[0] + v0 * p.vcs[1] + row * p.vcs[2] + c0 * p.vcs[3],
         p.vcs[1], p.vs[3], p.vcs[3], v1 - v0, false);
  }
}

static void bytes_of(long long* to, const int64_t* strides, int es) {
  for (int d = 0; d < 4; ++d) to[d] = (long long)strides[d] * es;
}

template <class T, bool kAppend>
static cudaError_t launch_rotate(RotateP& p, int vec, bool paired, cudaStream_t st) {
  const int per_thread = paired ? (vec == 1 ? 2 : vec) : vec;  // channels of a thread's pairs, counted on one side of a pair
  p.turning = (paired ? 2 * p.pairs : p.pairs) / per_thread;
  p.per_row = p.turning + (p.D - 2 * p.pairs) / vec;
  const long long items = (long long)p.B * p.L * p.per_row;
  p.items = (unsigned)items;
  const int per_block = vec * (int)sizeof(T) == 16 ? 32 : kThreads, shares = kThreads / per_block;  // kItems
  const long long blocks = (items + per_block - 1) / per_block;
  // Heads in as many slices as fill the SMs with 8 blocks each (4 prompts of 1000 tokens, 24 and 8 heads of 128: 18.7 us, with 16 19.0); a block has `shares` of them
  const long long want = 8ll * sm_count();
  const long long more = blocks >= want ? 1 : (want + blocks - 1) / blocks;
  const dim3 grid((unsigned)blocks, (unsigned)imax(1, imin((int)more, (p.heads + shares - 1) / shares)));
  p.slices = (int)grid.y * shares;
#define CHILL_ROTATE(VEC)                                                     \
  case VEC:                                                                   \
    if (paired) rotate_kernel<T, VEC, true, kAppend><<<grid, kThreads, 0, st>>>(p); \
    else rotate_kernel<T, VEC, false, kAppend><<<grid, kThreads, 0, st>>>(p);       \
    break
  switch (vec) {
    CHILL_ROTATE(1);
    CHILL_ROTATE(2);
    CHILL_ROTATE(4);
    default:
      if constexpr (sizeof(T) == 2) {
        if (paired) rotate_kernel<T, 8, true, kAppend><<<grid, kThreads, 0, st>>>(p);
        else rotate_kernel<T, 8, false, kAppend><<<grid, kThreads, 0, st>>>(p);
      }
  }
#undef CHILL_ROTATE
  return cudaGetLastError();
}

static int rotate(const chill_rotate_args* a, bool append, cudaStream_t st) {
  if (a == nullptr || a->B <= 0 || a->L <= 0 || a->D <= 0 || a->pairs <= 0 || a->pairs > a->D / 2 || a->n_axes <= 0) return CHILL_E_INVALID;
  if (!known_dtype(a->dtype)) return CHILL_E_UNSUPPORTED;
  if (!a->inv_freq || !a->positions) return CHILL_E_INVALID;
  if ((a->interleaved | a->inverse) & ~1) return CHILL_E_INVALID;
  if (a->q == nullptr && a->k == nullptr) return CHILL_E_INVALID;
  if ((a->q == nullptr) != (a->q_out == nullptr) || (!append && (a->k == nullptr) != (a->k_out == nullptr))) return CHILL_E_INVALID;
  if ((a->q != nullptr && a->H <= 0) || (a->k != nullptr && a->H_kv <= 0)) return CHILL_E_INVALID;
  if (append) {
    if (!a->q || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->slots || a->num_pages <= 0 || a->page_size <= 0 || a->inverse) return CHILL_E_INVALID;
    if ((long long)a->num_pages * a->page_size > 0x7fffffffll) return CHILL_E_TOO_LARGE;
  }
  if ((long long)a->B * a->L > 0x7fffffffll || (long long)a->B * a->L * a->D > 0x7fffffffll || a->H > (1 << 20) || a->H_kv > (1 << 20)) return CHILL_E_TOO_LARGE;
  RotateP p{};
  p.B = a->B; p.L = a->L; p.D = a->D; p.pairs = a->pairs; p.n_axes = a->n_axes; p.inverse = a->inverse;
  p.H = a->q != nullptr ? a->H : 0;
  p.Hkv = a->k != nullptr ? a->H_kv : 0;
  p.heads = p.H + p.Hkv * (append ? 2 : 1);
  p.inv_freq = a->inv_freq; p.axes = a->axes; p.positions = a->positions;
  p.pos_axis = a->position_strides[0]; p.pos_batch = a->position_strides[1]; p.pos_token = a->position_strides[2];
  p.q = (const char*)a->q; p.k = (const char*)a->k; p.v = (const char*)a->v;
  p.qo = (char*)a->q_out; p.ko = (char*)a->k_out; p.kc = (char*)a->k_cache; p.vc = (char*)a->v_cache;
  p.slots = a->slots; p.num_pages = a->num_pages; p.page = a->page_size;
  const int es = elem_size(a->dtype);
  int vec = 16 / es;
  auto uses = [&](const void* ptr, const int64_t* strides, long long* to) {
    if (ptr == nullptr) return;
    vec = imin(vec, row_vector(ptr, strides, 3, es) / es);
    bytes_of(to, strides, es);
  };
  uses(a->q, a->q_strides, p.qs);
  uses(a->k, a->k_strides, p.ks);
  if (p.H) uses(a->q_out, a->q_out_strides, p.qos);
  if (append) {
    uses(a->v, a->v_strides, p.vs);
    uses(a->k_cache, a->k_cache_strides, p.kcs);
    uses(a->v_cache, a->v_cache_strides, p.vcs);
  } else if (p.Hkv) {
    uses(a->k_out, a->k_out_strides, p.kos);
  }
  // A vector lies on one side of the pairs, or among the channels that stay
  while (vec > 1 && (a->D % vec != 0 || (a->interleaved ? 2 * a->pairs : a->pairs) % vec != 0)) vec /= 2;
  cudaError_t e;
#define CHILL_ROTATE_TYPE(T) e = append ? launch_rotate<T, true>(p, vec, a->interleaved != 0, st) : launch_rotate<T, false>(p, vec, a->interleaved != 0, st)
  if (a->dtype == CHILL_F32) CHILL_ROTATE_TYPE(float);
  else if (a->dtype == CHILL_F16) CHILL_ROTATE_TYPE(__half);
  else CHILL_ROTATE_TYPE(__nv_bfloat16);
#undef CHILL_ROTATE_TYPE
  if (e != cudaSuccess) return record_cuda_failure(e, "rotate launch");
  count_launches(1);
  return CHILL_OK;
}

}  // namespace decode
}  // namespace chill

extern "C" {

int chill_rotate(const chill_rotate_args* a, void* stream) { return chill::decode::rotate(a, false, (cudaStream_t)stream); }
int chill_rotate_append(const chill_rotate_args* a, void* stream) { return chill::decode::rotate(a, true, (cudaStream_t)stream); }

}  // extern "C"
