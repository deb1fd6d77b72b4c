// Selection of a beam search (chill_beam_select, include/chill_decode.h): candidates c = s_k + x_kv - lse_k of the K beams of a group over a vocabulary of V,
// the M largest of them.
//
// The logits are read once, and that is the floor.  Within a row the order is that of x, so while a warp streams its segment of a row it keeps the M
// largest x beside the running maximum and sum of the softmax, without knowing lse yet.  A cluster has a group: its warps share the rows, exchange maxima and
// sums through distributed shared memory, and only then turn their lists into candidates, which are merged by warps, CTAs and at last by the
// cluster's first CTA.  One launch, no workspace.
//
// A list is sorted and lies across the lanes of a warp (64 entries: two a lane).  What beats its last entry is collected in shared memory and merged in 32
// or 64 at a time by a bitonic network: the threshold lags behind by a batch, but a batch costs about 150 instructions where single insertions cost 25
// each, and a threshold of the M-th largest of t values lets about M of the next t through, so a segment of n values has log2(n / M) batches.
#include <cooperative_groups.h>

#include <type_traits>

#include "decode_common.cuh"

namespace chill {
namespace decode {
namespace cg = cooperative_groups;

struct SelectP {
  int K, M, V, per_row;  // per_row: warps (segments) of a row
  int segment;           // values of a segment, whole vectors
  const void* logits;
  long long row_stride;
  const float* scores;
  const uint8_t* finished;
  int end_token;
  float* out_scores;
  int *out_rows, *out_tokens;
};

constexpr int kWarps = 8;
constexpr int kMaxCluster = 16;
constexpr int kMost = CHILL_SELECT_MAX;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ long long imin64(long long a, long long b) { return a < b ? a : b; }

// A value and its place as one number: larger values first, of equal ones the lower place.  0: nothing (NaN never gets in).
__device__ __forceinline__ uint64_t key_of(float x, int v) {
  const uint32_t bits = __float_as_uint(x + 0.f);  // -0 is 0
  const uint32_t up = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
  return ((uint64_t)up << 32) | (uint32_t)~v;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up ^ 0x80000000u : ~up);
}
__device__ __forceinline__ int place_of(uint64_t key) { return (int)~(uint32_t)key; }

// A candidate: its 64-bit value mapped to a whole number in the same order (NaN on top), then the place among the group's K * V.  rank 0: nothing.
struct Candidate {
  uint64_t rank, place;  // place: inverted, larger is earlier
};
__device__ __forceinline__ uint64_t rank_of(double c) {
  if (c != c) return ~0ull;
  const uint64_t bits = (uint64_t)__double_as_longlong(c + 0.0);
  return bits ^ ((uint64_t)((int64_t)bits >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of_rank(uint64_t rank) {
  if (rank == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)(rank & 0x8000000000000000ull ? rank ^ 0x8000000000000000ull : ~rank));
}

__device__ __forceinline__ bool before(uint64_t a, uint64_t b) { return a > b; }
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.rank != b.rank ? a.rank > b.rank : a.place > b.place; }
__device__ __forceinline__ uint64_t from_lane(uint64_t x, int mask) { return __shfl_xor_sync(0xffffffffu, x, mask); }
__device__ __forceinline__ Candidate from_lane(const Candidate& x, int mask) {
  return {__shfl_xor_sync(0xffffffffu, x.rank, mask), __shfl_xor_sync(0xffffffffu, x.place, mask)};
}

// Lists of 32 * R entries over a warp: entry e is in register e / 32 of lane e % 32.  Sorted: entry 0 comes first.
template <class T, int R>
struct List {
  T x[R];

  // Entry e takes the earlier of e and e ^ distance where `keep_first` says so of it, else the later.
  __device__ __forceinline__ void step(int distance, int block) {
    const int lane = threadIdx.x & 31;
    if (R == 2 && distance == 32) {  // only for block 64, which is one direction
      const bool swap = before(x[R - 1], x[0]);
      const T a = x[0], b = x[R - 1];
      x[0] = swap ? b : a;
      x[R - 1] = swap ? a : b;
      return;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = lane + 32 * r;
      const T other = from_lane(x[r], distance);
      const bool first = ((e & distance) == 0) == ((e & block) == 0);
      if (before(other, x[r]) == first) x[r] = other;
    }
  }
  // A bitonic sequence becomes sorted.
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int distance = 16 * R; distance > 0; distance >>= 1) step(distance, 0);
  }
  __device__ __forceinline__ void sort() {
#pragma unroll
    for (int block = 2; block < 32 * R; block <<= 1)
#pragma unroll
      for (int distance = block >> 1; distance > 0; distance >>= 1) step(distance, block);
    settle();
  }
  // The 32 * R first of this list and of another one, given from its last entry to its first (entry e of `reversed` is entry 32 * R - 1 - e).
  __device__ __forceinline__ void merge(const List& reversed) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (before(reversed.x[r], x[r])) x[r] = reversed.x[r];
    settle();
  }
};


__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest number below x (x finite); what is above it is at least x.
__device__ __forceinline__ float just_below(float x) {
  const int bits = __float_as_int(x);
  return x == 0.f ? __int_as_float((int)0x80000001u) : __int_as_float(x > 0.f ? bits - 1 : bits + 1);
}

// What a warp knows of the segment that it streams.
template <int R>
struct Stream {
  List<uint64_t, R> best;
  float top;   // of this lane's values; their sum of exponentials relative to it, in 64 bits (a vector's terms are added up before)
  double sum;
  uint64_t* waiting;
  int count;    // of those that wait
  float limit;  // what is not above it is not among the M largest
  int last;     // M - 1

  __device__ __forceinline__ void begin(uint64_t* buffer, int M) {
#pragma unroll
    for (int r = 0; r < R; ++r) best.x[r] = 0;
    top = -INFINITY;
    sum = 0.0;
    waiting = buffer;
    count = 0;
    limit = -INFINITY;
    last = M - 1;
  }

  // Merges the first 32 * R that wait (what is missing of them is nothing) and moves the rest to the front.
  __device__ __forceinline__ void flush() {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    List<uint64_t, R> more, reversed;
#pragma unroll
    for (int r = 0; r < R; ++r) more.x[r] = lane + 32 * r < count ? waiting[lane + 32 * r] : 0;
    more.sort();
#pragma unroll
    for (int r = 0; r < R; ++r) reversed.x[r] = __shfl_sync(0xffffffffu, more.x[R - 1 - r], 31 - lane);
    best.merge(reversed);
    const uint64_t key = __shfl_sync(0xffffffffu, last >= 32 ? best.x[R - 1] : best.x[0], last & 31);
    if (key != 0) limit = value_of(key);
    const int rest = count - 32 * R;
    for (int e0 = 0; e0 < rest; e0 += 32) {
      const uint64_t x = e0 + lane < rest ? waiting[32 * R + e0 + lane] : 0;
      __syncwarp();
      if (e0 + lane < rest) waiting[e0 + lane] = x;
      __syncwarp();
    }
    count = imax(rest, 0);
  }

  // A lower limit to begin with: the M-th largest of 32 * R values, each the maximum of values of its own.
  __device__ __forceinline__ void first_limit(const float (&maxima)[R]) {
    List<uint64_t, R> sample;
#pragma unroll
    for (int r = 0; r < R; ++r) sample.x[r] = key_of(maxima[r], 0);
    sample.sort();
    const float found = value_of(__shfl_sync(0xffffffffu, last >= 32 ? sample.x[R - 1] : sample.x[0], last & 31));
    if (found > -INFINITY) limit = just_below(found);
  }

  // N values of each lane, the first of them number v of the row; -inf where there is none.
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float most) {
    if (most > top) {
      sum *= (double)exp2_of((top - most) * kLog2e);  // 0 * 0 the first time
      top = most;
    }
    const float base = top == -INFINITY ? 0.f : top;  // nothing but -inf so far
    float terms = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) terms += exp2_of((x[e] - base) * kLog2e);
    sum += (double)terms;
  }
  // Those above the limit wait; flush() has to follow where 32 * R do.
  template <int N>
  __device__ __forceinline__ void keep(const float (&x)[N], int v) {
    const unsigned below = (1u << (threadIdx.x & 31)) - 1;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool in = x[e] > limit;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      if (in) waiting[count + __popc(who & below)] = key_of(x[e], v + e);
      count += __popc(who);
    }
  }
};

template <class T, int V>
__device__ __forceinline__ float unpack(const uint4& raw, float (&x)[V]) {
  const T* p = reinterpret_cast<const T*>(&raw);
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    x[e] = Elem<T>::up(p[e]);
    most = fmaxf(most, x[e]);  // without NaN; these show in the sum
  }
  return most;
}

// 16 bytes from `byte` bytes into the first of two adjacent vectors on (a multiple of the element size).
__device__ __forceinline__ uint4 straddle(const uint4& a, const uint4& b, int byte) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t x[5];  // from the word on that the byte lies in
#pragma unroll
  for (int i = 0; i < 5; ++i) x[i] = byte < 4 ? w[i] : (byte < 8 ? w[i + 1] : (byte < 12 ? w[i + 2] : w[i + 3]));
  const int bits = 8 * (byte & 3);
  return make_uint4(__funnelshift_r(x[0], x[1], bits), __funnelshift_r(x[1], x[2], bits), __funnelshift_r(x[2], x[3], bits), __funnelshift_r(x[3], x[4], bits));
}

// Values [from, to) of a row, `from` a whole number of vectors of 16 bytes: a lane has a vector at a time, the last few values come at the end.  Which value is whose
// depends on its number alone, not on where the row lies in memory: equal rows have equal sums to the last bit, so that equal beams are ties.
// kShifted: rows do not begin at multiples of 16 bytes; a vector is put together from the two that it lies in, the first and the last one of a segment, whose
// neighbours are another's, value by value.
template <class T, int R, bool kShifted>
__device__ __forceinline__ void stream_row(Stream<R>& s, const T* row, int from, int to) {
  constexpr int V = 16 / sizeof(T), kBatch = kShifted ? 2 : 4;
  const int lane = threadIdx.x & 31, vectors = (to - from) / V;
  const int byte = kShifted ? (int)(reinterpret_cast<uintptr_t>(row) % 16) : 0;
  const uint4* at = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row + from) - byte);
  // -inf in every element, where there is no vector
  const uint32_t none = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u);
  for (int n0 = 0; n0 < vectors; n0 += 32 * kBatch) {
    uint4 raw[kBatch];
    float most[kBatch], x[V];
    if constexpr (kShifted) {
      uint4 next[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int n = n0 + 32 * u + lane;
        raw[u] = next[u] = make_uint4(none, none, none, none);
        if (n > 0 && n < vectors - 1) {
          raw[u] = __ldg(at + n);
          next[u] = __ldg(at + n + 1);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int n = n0 + 32 * u + lane;
        raw[u] = straddle(raw[u], next[u], byte);
        if (n == 0 || n == vectors - 1) {
          T* to_raw = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
          for (int e = 0; e < V; ++e) to_raw[e] = row[from + n * V + e];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int n = n0 + 32 * u + lane;
        raw[u] = n < vectors ? __ldcs(at + n) : make_uint4(none, none, none, none);
      }
    }
    float block = -INFINITY;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      most[u] = unpack<T, V>(raw[u], x);
      s.add(x, most[u]);
      block = fmaxf(block, most[u]);
    }
    if (n0 == 0) {
      float maxima[R];
#pragma unroll
      for (int r = 0; r < R; ++r) maxima[r] = -INFINITY;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) maxima[u % R] = fmaxf(maxima[u % R], most[u]);
      s.first_limit(maxima);
    }
    if (!__any_sync(0xffffffffu, block > s.limit)) continue;
#pragma unroll 1
    for (int u = 0; u < kBatch; ++u) {
      uint4 one = raw[0];
#pragma unroll
      for (int i = 1; i < kBatch; ++i) one = u == i ? raw[i] : one;
      if (!__any_sync(0xffffffffu, unpack<T, V>(one, x) > s.limit)) continue;
      s.keep(x, from + (n0 + 32 * u + lane) * V);
      while (s.count >= 32 * R) s.flush();
    }
  }
  const int v = from + vectors * V + lane;
  const float x[1] = {v < to ? Elem<T>::up(row[v]) : -INFINITY};
  s.add(x, fmaxf(x[0], -INFINITY));
  s.keep(x, v);
  while (s.count > 0) s.flush();
}

template <class T, int R, bool kShifted>
__global__ void __launch_bounds__(kWarps * 32) select_kernel(const __grid_constant__ SelectP p) {
  constexpr int kList = 32 * R, kBuffer = kList + 32 * (16 / (int)sizeof(T));
  union Room {  // of a warp: what waits while it streams, its list of candidates later
    uint64_t waiting[kBuffer];
    Candidate list[kList];
  };
  __shared__ __align__(16) unsigned char room_bytes[kWarps * sizeof(Room)];
  __shared__ __align__(16) unsigned char list_bytes[kMaxCluster * kList * sizeof(Candidate)];  // first CTA: the lists of all
  __shared__ float tops[kWarps];
  __shared__ double sums[kWarps];
  Room* const room = reinterpret_cast<Room*>(room_bytes);
  Candidate(*const lists)[kList] = reinterpret_cast<Candidate(*)[kList]>(list_bytes);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank(), group = (int)blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Unit u of the cluster, segment u % per_row of beam u / per_row, is warp u / ctas of CTA u % ctas
  const int unit = warp * ctas + cta, k = unit / p.per_row, part = unit - k * p.per_row;
  const bool works = k < p.K;
  const float base = works ? p.scores[group * p.K + k] : -INFINITY;
  const bool over = works && p.finished != nullptr && p.finished[group * p.K + k] != 0;
  const bool reads = works && !over && base != -INFINITY;
  const T* row = reinterpret_cast<const T*>(p.logits) + (long long)(group * p.K + k) * p.row_stride;
  Stream<R> s;
  s.begin(room[warp].waiting, p.M);
  if (reads) {
    const int from = (int)imin64((long long)part * p.segment, p.V), to = (int)imin64((long long)(part + 1) * p.segment, p.V);
    if (from < to) stream_row<T, R, kShifted>(s, row, from, to);
  }
  float top = s.top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  double sum = s.top == -INFINITY ? s.sum : s.sum * exp((double)s.top - (double)top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    tops[warp] = top;
    sums[warp] = sum;
  }
  cluster.sync();

  // log sum exp of the row, from all its segments
  List<Candidate, R> mine;
#pragma unroll
  for (int r = 0; r < R; ++r) mine.x[r] = {0, 0};
  if (reads) {
    float all = -INFINITY;
    double total = 0.0;
    for (int u = k * p.per_row + lane; u < (k + 1) * p.per_row; u += 32) all = fmaxf(all, *cluster.map_shared_rank(&tops[u / ctas], u % ctas));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
    for (int u = k * p.per_row + lane; u < (k + 1) * p.per_row; u += 32) {
      const float t = *cluster.map_shared_rank(&tops[u / ctas], u % ctas);
      const double x = *cluster.map_shared_rank(&sums[u / ctas], u % ctas);
      total += t == -INFINITY ? x : x * exp((double)t - (double)all);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const double lse = (double)all + log(total);
    const long long first = (long long)k * p.V;
    auto candidate = [&](float x, int v) { return Candidate{rank_of((double)base + ((double)x - lse)), ~(uint64_t)(first + v)}; };
    if (lse != lse || base != base || base == INFINITY) {
      // All candidates are equal (NaN, or +inf): the first ones count
      if (part == 0) {
        int found = 0;
        for (int v0 = 0; v0 < p.V && found < p.M; v0 += 32) {
          const float x = v0 + lane < p.V ? Elem<T>::up(row[v0 + lane]) : -INFINITY;
          const unsigned who = __ballot_sync(0xffffffffu, x != -INFINITY);
          const int e = found + __popc(who & ((1u << lane) - 1));
          if (x != -INFINITY && e < kList) room[warp].list[e] = candidate(x, v0 + lane);
          found += __popc(who);
        }
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (lane + 32 * r < found) mine.x[r] = room[warp].list[lane + 32 * r];
        __syncwarp();
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (s.best.x[r] != 0) mine.x[r] = candidate(value_of(s.best.x[r]), place_of(s.best.x[r]));
    }
  } else if (over && part == 0 && base != -INFINITY && lane == 0) {
    mine.x[0] = {rank_of((double)base), ~(uint64_t)((long long)k * p.V + p.end_token)};
  }

  // The lists of the warps, two and two
  auto merge_with = [&](const Candidate* list) {
    List<Candidate, R> reversed;
#pragma unroll
    for (int r = 0; r < R; ++r) reversed.x[r] = list[kList - 1 - lane - 32 * r];
    mine.merge(reversed);
  };
  auto merge_warps = [&]() {
#pragma unroll
    for (int apart = 1; apart < kWarps; apart <<= 1) {
      if ((warp & (2 * apart - 1)) == apart) {
#pragma unroll
        for (int r = 0; r < R; ++r) room[warp].list[lane + 32 * r] = mine.x[r];
      }
      __syncthreads();
      if ((warp & (2 * apart - 1)) == 0) merge_with(room[warp + apart].list);
    }
  };
  merge_warps();
  if (ctas > 1) {
    if (warp == 0) {
      Candidate* to = cluster.map_shared_rank(&lists[cta][0], 0);
#pragma unroll
      for (int r = 0; r < R; ++r) to[lane + 32 * r] = mine.x[r];
    }
    cluster.sync();
    if (cta != 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) mine.x[r] = warp < ctas ? lists[warp][lane + 32 * r] : Candidate{0, 0};
    if (warp + kWarps < ctas) merge_with(lists[warp + kWarps]);
    __syncthreads();  // room is written again
    merge_warps();
  }
  if (warp != 0) return;

  // Fewer than M that are not -inf: these are all there are, and the others follow in the order of their places
  int found = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    found += __popc(__ballot_sync(0xffffffffu, mine.x[r].rank != 0));
    room[0].list[lane + 32 * r] = mine.x[r];
  }
  __syncwarp();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = lane + 32 * r;
    if (e >= p.M) continue;
    long long place = (long long)~mine.x[r].place;
    double value = -INFINITY;
    if (e < found) {
      value = value_of_rank(mine.x[r].rank);
    } else {
      long long before_it = -1, places = 0;  // of those found
      while (places != before_it) {
        before_it = places;
        places = 0;
        for (int n = 0; n < found; ++n) places += (long long)~room[0].list[n].place <= e - found + before_it;
      }
      place = e - found + places;
    }
    const long long at = (long long)group * p.M + e;
    const int beam = (int)(place / p.V);
    p.out_scores[at] = (float)value;
    p.out_rows[at] = group * p.K + beam;
    p.out_tokens[at] = (int)(place - (long long)beam * p.V);
  }
}

template <class T, int R, bool kShifted>
static cudaError_t launch_kernel(const SelectP& p, int groups, int ctas, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  if (ctas > 8) {
    const cudaError_t e = cudaFuncSetAttribute(select_kernel<T, R, kShifted>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cfg.gridDim = dim3((unsigned)(groups * ctas));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, select_kernel<T, R, kShifted>, p);
}

template <class T>
static cudaError_t launch_select(const SelectP& p, int groups, int ctas, cudaStream_t st) {
  const bool shifted = reinterpret_cast<uintptr_t>(p.logits) % 16 != 0 || (groups * p.K > 1 && p.row_stride * (long long)sizeof(T) % 16 != 0);
  if (p.M <= 32) return shifted ? launch_kernel<T, 1, true>(p, groups, ctas, st) : launch_kernel<T, 1, false>(p, groups, ctas, st);
  return shifted ? launch_kernel<T, 2, true>(p, groups, ctas, st) : launch_kernel<T, 2, false>(p, groups, ctas, st);
}

static int select(const chill_select_args* a, cudaStream_t st) {
  if (a == nullptr || a->G <= 0 || a->K <= 0 || a->M <= 0 || a->V <= 0) return CHILL_E_INVALID;
  if (!known_dtype(a->dtype)) return CHILL_E_UNSUPPORTED;
  if (a->K > kMost || a->M > kMost || a->V > (1ll << 30) || (long long)a->G * a->K > kMaxRequests) return CHILL_E_TOO_LARGE;
  if (a->M > a->K * a->V || !a->logits || !a->scores || !a->out_scores || !a->out_rows || !a->out_tokens) return CHILL_E_INVALID;
  if (a->finished != nullptr && (a->end_token < 0 || a->end_token >= a->V)) return CHILL_E_INVALID;
  SelectP p{};
  p.K = a->K; p.M = a->M; p.V = (int)a->V;
  p.logits = a->logits; p.row_stride = a->row_stride;
  p.scores = a->scores; p.finished = a->finished; p.end_token = (int)a->end_token;
  p.out_scores = a->out_scores; p.out_rows = a->out_rows; p.out_tokens = a->out_tokens;
  // A warp for every beam at least; more CTAs while they fit the GPU, four an SM, and a warp has a thousand values
  int ctas = 1;
  while (ctas * kWarps < a->K) ctas *= 2;
  while (ctas < kMaxCluster && 2ll * ctas * a->G <= 4ll * sm_count() && (long long)a->K * a->V >= 2ll * ctas * kWarps * 1024) ctas *= 2;
  p.per_row = ctas * kWarps / a->K;
  const int vec = 16 / elem_size(a->dtype);
  const long long segment = (a->V + p.per_row - 1) / p.per_row;
  p.segment = (int)((segment + vec - 1) / vec * vec);
  cudaError_t e;
  if (a->dtype == CHILL_F32) e = launch_select<float>(p, a->G, ctas, st);
  else if (a->dtype == CHILL_F16) e = launch_select<__half>(p, a->G, ctas, st);
  else e = launch_select<__nv_bfloat16>(p, a->G, ctas, st);
  if (e != cudaSuccess) return record_cuda_failure(e, "select launch");
  count_launches(1);
  return CHILL_OK;
}

}  // namespace decode
}  // namespace chill

extern "C" int chill_beam_select(const chill_select_args* a, void* stream) { return chill::decode::select(a, (cudaStream_t)stream); }
