// Selection of a beam search (chill_beam_select, include/chill_decode.h): candidates c = s_k + x_kv - lse_k of the K beams of a group over a vocabulary of V,
// the M largest of them.
//
// The logits are read once, and that is the floor.  Within a row the order is that of x, so a CTA that streams a segment of a row keeps the M largest x beside the
// maximum and sum of the softmax, without knowing lse yet; a second kernel, a CTA for each group, turns the segments' lists into candidates and merges them.  Replayed from a
// graph: 32 groups of 8 beams over 128000 tokens in bf16, 16 candidates 30 us (floor 9), 4 groups of 32 beams over 50021 in fp32, 64 candidates 27 us (floor 4), one group of 4 beams
// over 32000 in fp32 10 us (floor: two launches).  One kernel with a group in a cluster of 16 CTAs, which exchange sums and lists through distributed shared memory, takes
// 62, 75 and 14 us: 64 CTAs do not fill the GPU, and lists that are kept sorted while they grow cost more than the logits.
//
// What is kept is not sorted while it grows.  The first batch of a segment gives a lower limit: a number that M of the 256 threads' maxima reach.  That
// lets about 1.5 M of 8192 values through; they wait in shared memory, where the limit is raised if they become many, and are sorted at the end.  Where more come than there is room
// for (sorted rows, constant ones) the M-th largest of all 256 thread maxima is a limit that leaves values of M threads.
#include <type_traits>

#include "decode_common.cuh"

namespace chill {
namespace decode {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMost = CHILL_SELECT_MAX;
constexpr int kBatch = 4;       // vectors of 16 bytes that a thread has at a time
constexpr int kMaxParts = 64;   // segments of a row
constexpr int kRoom = 2304;     // values that wait: those of M threads and more, a whole number for each thread
constexpr int kQueue = 96;       // vectors of a warp that wait to be looked at, after so many batches that 36 are to be expected (M = 64)
constexpr float kLog2e = 1.4426950408889634f;

struct Sum {
  double sum;
  float top;
  int padding;
};

struct SelectP {
  int K, M, V, parts;
  int segment;  // values of a segment, whole vectors
  const void* logits;
  long long row_stride;
  const float* scores;
  const uint8_t* finished;
  int end_token;
  uint64_t* lists;  // [row][part][M], descending
  Sum* sums;        // [row][part]
  float* out_scores;
  int *out_rows, *out_tokens;
};

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

// So many of what may be among the M largest are not worth another look at it.
__host__ __device__ constexpr int enough(int M) { return M + M / 4 + 1; }

// The order of numbers as 32 bits; nothing (-inf) is 0.
__device__ __forceinline__ uint32_t order_of(float x) { return x > -INFINITY ? (uint32_t)(key_of(x, 0) >> 32) : 0; }

// 64-bit scores in their order as whole numbers, NaN on top; 0: nothing.
__device__ __forceinline__ uint64_t rank_of(double c) {
  if (c != c) return ~0ull;
  const uint64_t bits = (uint64_t)__double_as_longlong(c + 0.0);
  return bits ^ ((uint64_t)((int64_t)bits >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of_rank(uint64_t rank) {
  if (rank == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double((long long)(rank & 0x8000000000000000ull ? rank ^ 0x8000000000000000ull : ~rank));
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The largest of 16 bytes of values; without NaN, these show in the sum.
template <class T>
__device__ __forceinline__ float vector_max(const uint4& raw) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(&raw);
    const T2 most = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(Elem<T>::up(most.x), Elem<T>::up(most.y));
  }
}

// Two fp32 numbers in one register pair: Blackwell adds and multiplies both in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split(uint64_t d, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// A candidate in the order of its 64-bit score, then of beam, logit and token, side by side and inverted (larger is earlier).  A row's list is in the order of the logits; 64 bits may
// round several of them to one score (a beam marked with -1e30), and the logit in the place leaves the list in order, which merging needs.
struct Candidate {
  uint64_t rank, place;
};
constexpr int kTokenBits = 26, kBeamBit = kTokenBits + 32;
static_assert(kMost <= 1 << (64 - kBeamBit), "a beam has too few bits");
__device__ __forceinline__ uint64_t place_at(int beam, uint32_t order, int token) {
  return ~((uint64_t)beam << kBeamBit | (uint64_t)~order << kTokenBits | (uint64_t)token);
}
__device__ __forceinline__ int beam_at(uint64_t place) { return (int)(~place >> kBeamBit); }
__device__ __forceinline__ int token_at(uint64_t place) { return (int)(~place & ((1u << kTokenBits) - 1)); }
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) { return a.rank != b.rank ? a.rank > b.rank : a.place > b.place; }

__device__ __forceinline__ bool before(uint64_t a, uint64_t b) { return a > b; }

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

// A segment's values that may be among its M largest, in shared memory.
struct alignas(16) Kept {
  uint64_t waiting[kRoom + 4];
  uint64_t maxima[kThreads];
  uint64_t nth;
  uint32_t least[kWarps], most[kWarps];
  int count;
  int queued[kWarps];
  uint4 queue[kWarps][kQueue];  // vectors in which a warp met something to keep, and their numbers
  int numbers[kWarps][kQueue];
};

// Every thread has a key, all that are not 0 are different: the M-th largest (0: there are fewer).
__device__ __forceinline__ uint64_t nth_of_threads(Kept& kept, uint64_t key, int M) {
  __syncthreads();
  kept.maxima[threadIdx.x] = key;
  if (threadIdx.x == 0) kept.nth = 0;
  __syncthreads();
  if (key != 0) {
    const ulonglong2* others = reinterpret_cast<const ulonglong2*>(kept.maxima);
    int larger = 0;
#pragma unroll 4
    for (int i = 0; i < kThreads / 2; ++i) larger += (others[i].x > key) + (others[i].y > key);
    if (larger == M - 1) kept.nth = key;
  }
  __syncthreads();
  return kept.nth;
}

// A number that at least M of the threads' numbers reach, and not many more, by halving (0: fewer than M are not 0; all alike: that one).  Some 8 barriers.
__device__ __forceinline__ uint32_t reached(Kept& kept, uint32_t own, int M) {
  const uint32_t least = __reduce_min_sync(0xffffffffu, own), largest = __reduce_max_sync(0xffffffffu, own);
  __syncthreads();  // what lies there has been read
  if ((threadIdx.x & 31) == 0) {
    kept.least[threadIdx.x >> 5] = least;
    kept.most[threadIdx.x >> 5] = largest;
  }
  __syncthreads();
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    lo = min(lo, kept.least[w]);
    hi = max(hi, kept.most[w]);
  }
  for (int i = 0; i < 20 && lo < hi; ++i) {
    const uint32_t middle = lo + (hi - lo) / 2 + 1;
    const int reach = __syncthreads_count(own >= middle);
    if (reach < M) {
      hi = middle - 1;
    } else {
      lo = middle;
      if (reach <= enough(M)) break;
    }
  }
  return lo > 0x007fffffu ? lo : 0;  // that is -inf
}

// Drops what is not among the M largest of those that wait until few more are left, a thread has one at most.  Returns how many; `limit` rises.
__device__ __forceinline__ int shrink(Kept& kept, int count, int M, uint64_t& limit) {
  bool exact = false;
  while (count > enough(M)) {
    uint64_t key[kRoom / kThreads], most = 0;
#pragma unroll
    for (int i = 0; i < kRoom / kThreads; ++i) {
      const int at = i * kThreads + (int)threadIdx.x;
      key[i] = at < count ? kept.waiting[at] : 0;
      most = key[i] > most ? key[i] : most;
    }
    const uint64_t lowest = exact ? nth_of_threads(kept, most, M) : (uint64_t)reached(kept, (uint32_t)(most >> 32), M) << 32;
    limit = lowest > limit ? lowest : limit;
    __syncthreads();
    if (threadIdx.x == 0) kept.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRoom / kThreads; ++i)
      if (key[i] != 0 && key[i] >= lowest) kept.waiting[atomicAdd(&kept.count, 1)] = key[i];
    __syncthreads();
    const int left = kept.count;
    __syncthreads();
    if (left == count) {  // many are alike: places decide
      if (count <= kThreads) break;
      exact = true;
    }
    count = left;
  }
  return count;
}

// Which value is whose depends on its number alone, not on where the row lies in memory: equal rows have equal sums to the last bit, so that equal beams are ties.
// A thread has vectors of 16 bytes; kShifted, where rows do not begin at multiples of 16 bytes: words of 4 bytes, 256 apart, of which rows that begin in the middle of one
// put theirs together from two.
//
// Warps stream on their own: sums in registers, vectors that reach the limit in a queue of their own, which are looked at value by value after a round of some batches.  32 groups of
// 8 beams over 128000 tokens, bf16: a segment's first batch and limit 4 us, the other seven 10 (5.8 TB/s), queue, sorting and sum 4; SMs with four CTAs are done 6 us after those with three.
// 128 threads a CTA, 8 of them an SM: 33 us instead of 30; half as long segments 31; the next batch's loads ahead of this one's work (3 CTAs an SM) no gain; the segment's rest prefetched into L2 31 to 33.
template <class T, bool kShifted>
__global__ void __launch_bounds__(kThreads, 4) scan_kernel(const __grid_constant__ SelectP p) {
  constexpr int V = 16 / sizeof(T), kWord = 4 / sizeof(T), kStep = kThreads * kBatch;
  __shared__ Kept kept;
  __shared__ Sum of_warps[kWarps];
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int beam = (int)blockIdx.x / p.parts, part = (int)blockIdx.x - beam * p.parts;
  const int from = part * p.segment, to = imin(from + p.segment, p.V);  // every segment has a value (parts_of)
  const T* row = reinterpret_cast<const T*>(p.logits) + beam * p.row_stride + from;
  const int size = to - from;
  if (p.scores[beam] == -INFINITY || (p.finished != nullptr && p.finished[beam] != 0)) return;  // nothing of it is looked at
  const uint32_t none = sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u);  // -inf in every element
  if (threadIdx.x == 0) kept.count = 0;
  float top = -INFINITY;  // of this thread's values; the sum of exponentials relative to it is kept in 64 bits, a batch's terms are added up before
  double sum = 0.0;
  uint64_t limit = 0;

  // kWord values from number v on, as far as they are there, the others -inf
  auto word_of = [&](int v) {
    uint32_t word = none;
    T* x = reinterpret_cast<T*>(&word);
#pragma unroll
    for (int e = 0; e < kWord; ++e)
      if (v + e < size) x[e] = row[v + e];
    return word;
  };
  // Number of element e of vector `id`: the first one of the batch + 256 u + thread
  auto number_of = [&](int id, int e) {
    if (!kShifted) return id * V + e;
    return (id / kStep * kStep * 4 + (id % kStep / kThreads * 4 + e / kWord) * kThreads + id % kThreads) * kWord + e % kWord;
  };
  auto load = [&](int n0, uint4 (&raw)[kBatch]) {
    const bool whole = n0 + kStep < size / V;  // every vector of the batch is there, and one more value
    if constexpr (kShifted) {
      uint32_t* words = reinterpret_cast<uint32_t*>(raw);
      const bool odd = reinterpret_cast<uintptr_t>(row) % 4 != 0;
      const uint32_t* at = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(row) / 4 * 4) + n0 * 4 + threadIdx.x;
      if (whole && sizeof(T) == 2 && odd) {
#pragma unroll
        for (int i = 0; i < 4 * kBatch; ++i) {
          if (i == 0 && n0 == 0 && threadIdx.x == 0) words[i] = word_of(0);  // half of the first word is another's
          else words[i] = __funnelshift_r(__ldg(at + i * kThreads), __ldg(at + i * kThreads + 1), 16);
        }
      } else if (whole && !(sizeof(T) == 2 && odd)) {
#pragma unroll
        for (int i = 0; i < 4 * kBatch; ++i) words[i] = __ldg(at + i * kThreads);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * kBatch; ++i) words[i] = word_of((n0 * 4 + i * kThreads + (int)threadIdx.x) * kWord);
      }
    } else {
      const uint4* at = reinterpret_cast<const uint4*>(row) + n0 + threadIdx.x;
      if (whole) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) raw[u] = __ldg(at + u * kThreads);
      } else {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int v = (n0 + u * kThreads + (int)threadIdx.x) * V;
          if (v + V <= size) raw[u] = __ldg(at + u * kThreads);
          else raw[u] = make_uint4(word_of(v), word_of(v + kWord), word_of(v + 2 * kWord), word_of(v + 3 * kWord));
        }
      }
    }
  };

  auto add_up = [&]() {  // a warp's sum, once it has streamed its part
    float highest = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, o));
    if (top != -INFINITY) sum *= (double)exp2_of((top - highest) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) of_warps[warp] = {sum, highest, 0};
  };
  const int round_step = imin(imax(192 / p.M, 1), 16) * kStep;
  for (int round = 0; round * V < size; round += round_step) {
    int queued = 0;
    const int end = imin(round + round_step, (size + V - 1) / V);
    for (int n0 = round; n0 < end; n0 += kStep) {
      uint4 raw[kBatch];
      load(n0, raw);
      float most[kBatch], all = -INFINITY;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        most[u] = vector_max<T>(raw[u]);
        all = fmaxf(all, most[u]);
      }
      if (all > top) {
        sum *= (double)exp2_of((top - all) * kLog2e);  // 0 * 0 the first time
        top = all;
      }
      const float base = top == -INFINITY ? 0.f : -top;  // nothing but -inf so far
      const uint64_t base2 = pair_of(base, base), log2e2 = pair_of(kLog2e, kLog2e);
      uint64_t terms = 0;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const T* x = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          float a, b;
          split(mul2(add2(pair_of(Elem<T>::up(x[e]), Elem<T>::up(x[e + 1])), base2), log2e2), a, b);
          terms = add2(terms, pair_of(exp2_of(a), exp2_of(b)));
        }
      }
      float even, uneven;
      split(terms, even, uneven);
      sum += (double)(even + uneven);

      if (n0 == 0) {
        limit = (uint64_t)reached(kept, order_of(all), p.M) << 32;
      }
      const float lowest = limit == 0 ? -INFINITY : value_of(limit);
      if (!__any_sync(0xffffffffu, all > -INFINITY && all >= lowest)) continue;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const unsigned who = __ballot_sync(0xffffffffu, most[u] > -INFINITY && most[u] >= lowest);
        const int at = queued + __popc(who & ((1u << lane) - 1));
        if ((who >> lane & 1) && at < kQueue) {
          kept.queue[warp][at] = raw[u];
          kept.numbers[warp][at] = n0 + u * kThreads + (int)threadIdx.x;
        }
        queued += __popc(who);
      }
    }
    if (lane == 0) kept.queued[warp] = queued;
    if (end * V >= size) add_up();
    __syncthreads();
    const int before = kept.count;
    int fullest = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) fullest = imax(fullest, kept.queued[w]);
    __syncthreads();
    if (fullest <= kQueue) {
      const float lowest = limit == 0 ? -INFINITY : value_of(limit);
      const T* values = reinterpret_cast<const T*>(kept.queue[warp]);
      for (int i = lane; i < queued * V; i += 32) {
        const float value = Elem<T>::up(values[i]);
        if (value > -INFINITY && value >= lowest) {
          const uint64_t key = key_of(value, from + number_of(kept.numbers[warp][i / V], i % V));
          if (key >= limit) {
            const int at = atomicAdd(&kept.count, 1);
            if (at < kRoom) kept.waiting[at] = key;
          }
        }
      }
      __syncthreads();
    }
    if (fullest > kQueue || kept.count > kRoom) {
      // Sorted or constant values, or very many that are alike: batch by batch, with the M-th largest of the threads' maxima as the limit, which leaves values of M threads
      __syncthreads();
      if (threadIdx.x == 0) kept.count = before;
      for (int n0 = round; n0 < end; n0 += kStep) {
        __syncthreads();
        shrink(kept, kept.count, p.M, limit);  // 256 wait at most
        uint4 raw[kBatch];
        load(n0, raw);
        uint64_t first = 0;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const T* x = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float value = Elem<T>::up(x[e]);
            const uint64_t key = value > -INFINITY ? key_of(value, from + number_of(n0 + u * kThreads + (int)threadIdx.x, e)) : 0;
            first = key > first ? key : first;
          }
        }
        const uint64_t nth = nth_of_threads(kept, first, p.M);
        limit = nth > limit ? nth : limit;
        if (first == 0 || first < limit) continue;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const T* x = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float value = Elem<T>::up(x[e]);
            const uint64_t key = value > -INFINITY ? key_of(value, from + number_of(n0 + u * kThreads + (int)threadIdx.x, e)) : 0;
            if (key != 0 && key >= limit) kept.waiting[atomicAdd(&kept.count, 1)] = key;
          }
        }
      }
    }
    if (end * V < size) {  // another round: its limit is about the M-th largest of those that wait
      __syncthreads();
      shrink(kept, kept.count, p.M, limit);
    }
  }

  __syncthreads();
  if (warp == 0) {
    const Sum s = of_warps[lane % kWarps];
    float highest = s.top;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, o));
    sum = s.top != -INFINITY ? s.sum * exp((double)s.top - (double)highest) : s.sum;
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) p.sums[blockIdx.x] = {sum, highest, 0};
  }
  // Its list.  A thread has a value at most: warps sort theirs, and a value's place is the sum of its places in all 8 sorted runs
  const int count = kept.count > kThreads ? shrink(kept, kept.count, p.M, limit) : kept.count;
  uint64_t* list = p.lists + (long long)blockIdx.x * p.M;
  List<uint64_t, 1> run;
  run.x[0] = (int)threadIdx.x < count ? kept.waiting[threadIdx.x] : 0;
  if (warp * 32 < count) run.sort();
  kept.maxima[threadIdx.x] = run.x[0];
  __syncthreads();
  const uint64_t key = run.x[0];
  if (key != 0) {
    int larger = lane;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint64_t* other = kept.maxima + w * 32;
      if (w == warp || w * 32 >= count || other[0] <= key) continue;
      int n = 0;  // how many of them are larger: between 1 and 32
#pragma unroll
      for (int step = 16; step > 0; step >>= 1) n += other[n + step - 1] > key ? step : 0;
      larger += n + (other[n] > key);
    }
    if (larger < p.M) list[larger] = key;
  }
  if ((int)threadIdx.x >= count && (int)threadIdx.x < p.M) list[threadIdx.x] = 0;
}

// One CTA for a group.  Up to 32 lists are merged two and two, by warps (bitonic networks).  Of more lists a lower limit, from their entries at some depths, leaves few candidates, which
// are sorted (4 groups of 32 beams in 4 segments, 64 candidates: 9 us, by merging 15; 32 groups of 8 beams in 2 segments, 16 candidates: 6 us, by merging 3).  Where very many are
// alike, or rows are NaN, many lists are merged too: a warp keeps the M first of those it has met, and merges a list of which the first entry comes before its last one.
constexpr int kMergeWarps = 32;  // at most: one for every list, and 4 at least
constexpr int kDepths = 7;       // 1, 2, 4, ... 64 entries
constexpr int kFound = 512;

template <class T, int R>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ SelectP p) {
  constexpr int kList = 32 * R;
  __shared__ double lse[kMost];
  __shared__ float score[kMost];
  __shared__ bool over[kMost], flat[kMost];  // finished beams; rows whose candidates are all alike: NaN or +inf
  __shared__ Candidate exchange[kMergeWarps / 2][kList], found[kFound];
  __shared__ uint32_t bounds[kDepths];
  __shared__ int n_found;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = (int)blockIdx.x, warps = (int)blockDim.x >> 5;
  const int lists = p.K * p.parts;
  const uint64_t* const entries = p.lists + (long long)group * lists * p.M;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the lists are there
  // Few lists: a warp has one, which is on its way while the sums are worked out (nonsense where nothing was written)
  const bool few = lists <= warps;
  uint64_t first[R];
#pragma unroll
  for (int r = 0; r < R; ++r) first[r] = few && warp < lists && lane + 32 * r < p.M ? __ldcg(&entries[(long long)warp * p.M + lane + 32 * r]) : 0;
  bool any_flat = false;
  for (int k = warp; k < p.K; k += warps) {
    const long long beam = (long long)group * p.K + k;
    const float s = p.scores[beam];
    const bool ended = p.finished != nullptr && p.finished[beam] != 0;
    Sum mine[kMaxParts / 32];  // nonsense for beams that were not looked at
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) mine[i] = lane + 32 * i < p.parts ? p.sums[beam * p.parts + lane + 32 * i] : Sum{0.0, -INFINITY, 0};
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) top = fmaxf(top, mine[i].top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i)
      if (lane + 32 * i < p.parts) sum += mine[i].top == -INFINITY ? mine[i].sum : mine[i].sum * exp((double)mine[i].top - (double)top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double l = (double)top + log(sum);  // a row without values has empty lists
    const bool alike = s != -INFINITY && !ended && (l != l || !(s < INFINITY));
    any_flat = any_flat || alike;
    if (lane == 0) {
      lse[k] = l;
      score[k] = s;
      over[k] = ended;
      flat[k] = alike;
    }
  }
  any_flat = __syncthreads_or(any_flat) != 0;
  auto candidate = [&](int k, float x, int v) {
    return Candidate{rank_of((double)score[k] + ((double)x - lse[k])), place_at(k, flat[k] ? 0 : order_of(x), v)};
  };
  auto usable = [&](int k) { return score[k] != -INFINITY && !over[k] && !flat[k]; };

  List<Candidate, R> best;
#pragma unroll
  for (int r = 0; r < R; ++r) best.x[r] = {0, 0};
  if (any_flat && warp < 2) {  // rows of NaN, rows of +inf: the first values of the first ones
    int n = 0;
    for (int k = 0; k < p.K; ++k) {
      if (!flat[k] || (score[k] == INFINITY && lse[k] == lse[k]) != (warp == 1)) continue;
      const T* row = reinterpret_cast<const T*>(p.logits) + ((long long)group * p.K + k) * p.row_stride;
      for (int v0 = 0; v0 < p.V && n < p.M; v0 += 32) {
        const float x = v0 + lane < p.V ? Elem<T>::up(row[v0 + lane]) : -INFINITY;
        const unsigned who = __ballot_sync(0xffffffffu, x != -INFINITY);
        const int e = n + __popc(who & ((1u << lane) - 1));
        if (x != -INFINITY && e < kList) exchange[warp][e] = candidate(k, x, v0 + lane);
        n += __popc(who);
      }
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane + 32 * r < n) best.x[r] = exchange[warp][lane + 32 * r];
  }

  // Entry e of list l
  auto entry = [&](int l, int e, uint64_t key) {
    const int k = l / p.parts;
    if (usable(k)) return key != 0 ? candidate(k, value_of(key), place_of(key)) : Candidate{0, 0};
    if (over[k] && e == 0 && l == k * p.parts && score[k] != -INFINITY)  // a finished beam: a list of one
      return Candidate{rank_of((double)score[k]), place_at(k, 0, p.end_token)};
    return Candidate{0, 0};
  };
  auto merge_all = [&]() {
    auto nth = [&]() {  // the M-th; with all lanes
      return Candidate{__shfl_sync(0xffffffffu, p.M > 32 ? best.x[R - 1].rank : best.x[0].rank, (p.M - 1) & 31),
                       __shfl_sync(0xffffffffu, p.M > 32 ? best.x[R - 1].place : best.x[0].place, (p.M - 1) & 31)};
    };
    if (warp < lists) {
      List<Candidate, R> own;
#pragma unroll
      for (int r = 0; r < R; ++r) own.x[r] = lane + 32 * r < p.M ? entry(warp, lane + 32 * r, few ? first[r] : entries[(long long)warp * p.M + lane + 32 * r]) : Candidate{0, 0};
      if (any_flat && warp < 2) {  // there may be something already: the list's entries from the last one to the first
        List<Candidate, R> reversed;
#pragma unroll
        for (int r = 0; r < R; ++r)
          reversed.x[r] = {__shfl_sync(0xffffffffu, own.x[R - 1 - r].rank, 31 - lane), __shfl_sync(0xffffffffu, own.x[R - 1 - r].place, 31 - lane)};
        best.merge(reversed);
      } else {
        best = own;
      }
    }
    for (int l0 = warp + warps; l0 < lists; l0 += 32 * warps) {  // of the others a lane looks at the first entry
      const int own = l0 + lane * warps;
      const Candidate head = own < lists ? entry(own, 0, entries[(long long)own * p.M]) : Candidate{0, 0};
      bool waits = head.rank != 0;
      while (true) {
        const Candidate last = nth();  // with all lanes
        waits = waits && before(head, last);
        // the one with the best first entry (or next to it), after which more are passed over
        const uint32_t top = waits ? (uint32_t)(head.rank >> 32) : 0, most = __reduce_max_sync(0xffffffffu, top);
        if (most == 0) break;
        const int next = __ffs(__ballot_sync(0xffffffffu, top == most)) - 1, l = l0 + next * warps;
        if (lane == next) waits = false;
        List<Candidate, R> reversed;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int e = kList - 1 - lane - 32 * r;
          reversed.x[r] = e < p.M ? entry(l, e, entries[(long long)l * p.M + e]) : Candidate{0, 0};
        }
        best.merge(reversed);
      }
    }
#pragma unroll 1
    for (int apart = warps / 2; apart > 0; apart >>= 1) {
      __syncthreads();  // what lies in `exchange` has been read
      if (warp >= apart && warp < 2 * apart) {
#pragma unroll
        for (int r = 0; r < R; ++r) exchange[warp - apart][lane + 32 * r] = best.x[r];
      }
      __syncthreads();
      if (warp < apart) {
        const Candidate last = nth();
        if (before(exchange[warp][0], last)) {
          List<Candidate, R> reversed;
#pragma unroll
          for (int r = 0; r < R; ++r) reversed.x[r] = exchange[warp][kList - 1 - lane - 32 * r];
          best.merge(reversed);
        }
      }
    }
  };
  // A lower limit.  Of n lists that have d entries each that reach a number, n d candidates do: for d = 1, 2, 4, ... the (M / d)-th largest of the lists' d-th entries, by their
  // leading 32 bits and by halving, and the largest of these numbers.  Some 1.3 M candidates reach it.
  bool by_limit = !few && !any_flat;
  if (by_limit && warp < kDepths) {
    const int depth = imin(1 << warp, p.M), need = (p.M + depth - 1) / depth;
    constexpr int kEach = 4;
    uint32_t x[kEach] = {};
    for (int l0 = lane; l0 < lists; l0 += 32 * kEach) {  // of more than 128 lists the largest of several
      uint64_t key[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) key[i] = l0 + 32 * i < lists ? __ldcg(&entries[(long long)(l0 + 32 * i) * p.M + depth - 1]) : 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (l0 + 32 * i < lists) x[i] = max(x[i], (uint32_t)(entry(l0 + 32 * i, depth - 1, key[i]).rank >> 32));
    }
    auto reach = [&](uint32_t number) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) n += __popc(__ballot_sync(0xffffffffu, x[i] >= number));
      return n;
    };
    uint32_t some = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kEach; ++i) some = x[i] != 0 ? min(some, x[i]) : some;
    uint32_t lo = __reduce_min_sync(0xffffffffu, some), hi = __reduce_max_sync(0xffffffffu, max(max(x[0], x[1]), max(x[2], x[3])));
    if (hi == 0 || reach(lo) < need) lo = hi = 0;  // fewer lists than that have so many entries
    while (lo < hi) {
      const uint32_t middle = lo + (hi - lo) / 2 + 1;
      const int n = reach(middle);
      if (n >= need) lo = middle;
      else hi = middle - 1;
      if (n >= need && n <= need + need / 8) break;
    }
    if (lane == 0) bounds[warp] = lo;
  }
  if (threadIdx.x == 0) n_found = 0;
  __syncthreads();
  uint32_t bound = 0;
#pragma unroll
  for (int i = 0; i < kDepths; ++i) bound = max(bound, bounds[i]);
  if (by_limit) {
    // A warp has a list at a time, a lane an entry (two); within a row the limit is one for the logits, rounded down
    const double least = value_of_rank((uint64_t)bound << 32);
    constexpr int kEach = 4;
    for (int l0 = warp; l0 < lists; l0 += warps * kEach) {
      uint64_t key[kEach][R];
#pragma unroll
      for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r)
          key[i][r] = l0 + i * warps < lists && lane + 32 * r < p.M ? __ldcg(&entries[(long long)(l0 + i * warps) * p.M + lane + 32 * r]) : 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int l = l0 + i * warps, k = l / p.parts;
        if (l >= lists) break;
        const double s = score[k], error = 1e-15 * (fabs(least) + fabs(s) + fabs(lse[k]));  // of the sum here and of the score's, 2^-53 each
        const float floor = bound == 0 ? -INFINITY : __double2float_rd(least - s + lse[k] - error);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool may = over[k] ? l == k * p.parts && lane == 0 && r == 0 : key[i][r] != 0 && !(value_of(key[i][r]) < floor);
          if (!may) continue;
          const Candidate c = entry(l, lane + 32 * r, key[i][r]);
          if (c.rank == 0 || (uint32_t)(c.rank >> 32) < bound) continue;
          const int at = atomicAdd(&n_found, 1);
          if (at < kFound) found[at] = c;
        }
      }
    }
  }
  __syncthreads();
  const int n = n_found;
  by_limit = by_limit && n <= kFound;
  if (by_limit) {
    // Runs of 32 are sorted; a candidate's place is the sum of its places in all of them
    for (int i0 = warp * 32; i0 < n; i0 += warps * 32) {
      List<Candidate, 1> run;
      run.x[0] = i0 + lane < n ? found[i0 + lane] : Candidate{0, 0};
      run.sort();
      found[i0 + lane] = run.x[0];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const Candidate c = found[i];
      int place = i & 31;
      for (int run = 0; run < n; run += 32) {
        if (run == (i & ~31) || !before(found[run], c)) continue;
        int larger = 0;
#pragma unroll
        for (int step = 16; step > 0; step >>= 1) larger += before(found[run + larger + step - 1], c) ? step : 0;
        place += larger + (before(found[run + larger], c) ? 1 : 0);
      }
      if (place < kList) exchange[1][place] = c;
    }
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int r = 0; r < R; ++r) best.x[r] = lane + 32 * r < n ? exchange[1][lane + 32 * r] : Candidate{0, 0};
  } else {
    // The lists are merged, two and two
    merge_all();
    if (warp != 0) return;
  }

  // Fewer than M that are not -inf: these are all there are, and the others follow in the order of their places
  int total = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    total += __popc(__ballot_sync(0xffffffffu, best.x[r].rank != 0));
    exchange[1][lane + 32 * r] = best.x[r];  // read by warp 1 in the last round but one
  }
  __syncwarp();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int e = lane + 32 * r;
    if (e >= p.M) continue;
    const long long to = (long long)group * p.M + e;
    int k = beam_at(best.x[r].place), v = token_at(best.x[r].place);
    double value = -INFINITY;
    if (e < total) {
      value = value_of_rank(best.x[r].rank);
    } else {
      long long so_far = -1, skipped = 0;  // of those found
      while (skipped != so_far) {
        so_far = skipped;
        skipped = 0;
        for (int i = 0; i < total; ++i) {
          const uint64_t place = exchange[1][i].place;
          skipped += (long long)beam_at(place) * p.V + token_at(place) <= e - total + so_far;
        }
      }
      k = (int)((e - total + skipped) / p.V);
      v = (int)(e - total + skipped - (long long)k * p.V);
    }
    p.out_scores[to] = (float)value;
    p.out_rows[to] = group * p.K + k;
    p.out_tokens[to] = v;
  }
}

// Segments of a row, and their length: whole batches, as many as the GPU has room for CTAs (four an SM).
static int parts_of(const chill_select_args& a, int& segment) {
  const int vec = 16 / elem_size(a.dtype), batch = kThreads * kBatch * vec;
  const long long batches = (a.V + batch - 1) / batch, rows = (long long)a.G * a.K, slots = 4ll * sm_count();
  long long parts = rows < slots ? slots / rows : 1;
  if (parts > kMaxParts) parts = kMaxParts;
  const long long each = (batches + parts - 1) / parts;
  segment = (int)(each * batch);
  return (int)((batches + each - 1) / each);
}

static size_t workspace_of(const chill_select_args& a) {
  int segment;
  const size_t lists = (size_t)a.G * a.K * parts_of(a, segment);
  return lists * (a.M * sizeof(uint64_t) + sizeof(Sum));
}

static int check_select(const chill_select_args* a, bool pointers) {
  if (a == nullptr || a->G <= 0 || a->K <= 0 || a->M <= 0 || a->V <= 0) return CHILL_E_INVALID;
  if (!known_dtype(a->dtype)) return CHILL_E_UNSUPPORTED;
  if (a->K > kMost || a->M > kMost || a->V > (1ll << kTokenBits) || (long long)a->G * a->K > kMaxRequests) return CHILL_E_TOO_LARGE;
  if (a->M > a->K * a->V) return CHILL_E_INVALID;
  if (!pointers) return CHILL_OK;
  if (!a->logits || !a->scores || !a->out_scores || !a->out_rows || !a->out_tokens) return CHILL_E_INVALID;
  if (a->finished != nullptr && (a->end_token < 0 || a->end_token >= a->V)) return CHILL_E_INVALID;
  if (a->workspace == nullptr || a->workspace_bytes < workspace_of(*a) || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0) return CHILL_E_INVALID;
  return CHILL_OK;
}

template <class T>
static cudaError_t launch_select(const SelectP& p, int groups, cudaStream_t st) {
  const bool shifted = reinterpret_cast<uintptr_t>(p.logits) % 16 != 0 || (groups * p.K > 1 && p.row_stride * (long long)sizeof(T) % 16 != 0);
  const unsigned units = (unsigned)(groups * p.K * p.parts);
  if (shifted) scan_kernel<T, true><<<units, kThreads, 0, st>>>(p);
  else scan_kernel<T, false><<<units, kThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // The second kernel is brought up beside the first one's last CTAs, and waits for their end (griddepcontrol)
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)groups);
  int warps = 4;
  while (warps < kMergeWarps && warps < p.K * p.parts) warps *= 2;
  cfg.blockDim = dim3(32u * (unsigned)warps);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return p.M <= 32 ? cudaLaunchKernelEx(&cfg, merge_kernel<T, 1>, p) : cudaLaunchKernelEx(&cfg, merge_kernel<T, 2>, p);
}

static int select(const chill_select_args& a, cudaStream_t st) {
  SelectP p{};
  p.K = a.K; p.M = a.M; p.V = (int)a.V;
  p.parts = parts_of(a, p.segment);
  p.logits = a.logits; p.row_stride = a.row_stride;
  p.scores = a.scores; p.finished = a.finished; p.end_token = (int)a.end_token;
  p.sums = (Sum*)a.workspace;
  p.lists = (uint64_t*)(p.sums + (size_t)a.G * a.K * p.parts);
  p.out_scores = a.out_scores; p.out_rows = a.out_rows; p.out_tokens = a.out_tokens;
  cudaError_t e;
  if (a.dtype == CHILL_F32) e = launch_select<float>(p, a.G, st);
  else if (a.dtype == CHILL_F16) e = launch_select<__half>(p, a.G, st);
  else e = launch_select<__nv_bfloat16>(p, a.G, st);
  if (e != cudaSuccess) return record_cuda_failure(e, "select launch");
  count_launches(2);
  return CHILL_OK;
}

}  // namespace decode
}  // namespace chill

extern "C" {

size_t chill_select_workspace_bytes(const chill_select_args* a) {
  return chill::decode::check_select(a, false) == CHILL_OK ? chill::decode::workspace_of(*a) : 0;
}

int chill_beam_select(const chill_select_args* a, void* stream) {
  const int st = chill::decode::check_select(a, true);
  return st != CHILL_OK ? st : chill::decode::select(*a, (cudaStream_t)stream);
}

}  // extern "C"
