// Log probabilities of given tokens, the entropy and the most probable alternatives of every row of logits, and their
// gradient.  With z = x / temperature, M = max x, S = sum exp((x - M) / temperature):
//
//   log p_j = (x_j - M) / temperature - log S
//   H       = log S - sum_j exp((x_j - M) / temperature) (x_j - M) / temperature / S
//   dx_j    = [ g_j - p_j (sum_i g_i + dH (log p_j + H)) ] / temperature
//
// where g is the gradient of the log probabilities: of the token's and of the alternatives', zero elsewhere.  M and log S
// are kept apart for the backward pass: their sum would lose the digits that small differences of logits are in.
#include "logprobs.h"

#include <cuda_bf16.h>

#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_PARTS = 8;
constexpr int AHEAD = 4;                 // vectors in flight per thread
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float FAR_BELOW = -1e30f;      // in place of -inf behind a subtraction: exp() of it is 0, and so is 0 times it

template <class T>
constexpr int VEC = 16 / sizeof(T);

// NaN where one of the two is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x to two units of the last place; results below the normal numbers are 0.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }

__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4], float) {
  f[0] = __uint_as_float(u.x);
  f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z);
  f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], __nv_bfloat16) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// ------------------------------------------------------------------ maximum and sums
// m = max x, s = sum 2^a, t = sum 2^a a, where a = (x - from) c2 and c2 = log2(e) / temperature.
struct Sums {
  float m, from, s, t;

  __device__ __forceinline__ static Sums none() { return {-INFINITY, -FLT_MAX, 0.f, 0.f}; }

  // All exponents `d` more.
  __device__ __forceinline__ void shift(float d) {
    const float f = ex2(d);
    t = f * fmaf(s, d, t);
    s *= f;
  }
  // The same sums from another, larger `from`.  With the row's maximum every term of t has one sign, so the entropy is a sum
  // without cancellation.
  __device__ __forceinline__ void rebase(float to, float c2) {
    shift(max_nan((from - to) * c2, FAR_BELOW));
    from = to;
  }
};

// What is not above `low`, a bf16 number of which low c2 is -2^30 or little above, has no weight in the quick pass.  Its exponents fma(x, c2,
// -base) keep what was lost when base = x c2 was rounded, half a unit of the last place: 64 at most for what is above low / 2, so a sum
// of a thread that has seen nothing but masked ids, whatever finite number they are masked by, is at most 2^64 times its length
// until it is brought to the row's maximum, beside which it is 0.  A row whose maximum is not inside (low / 2, -low / 2), or whose
// alternatives reach down to low, is read again by the exact pass.
float lowest_logit(float inv_t) {
  const float low = -1073741824.f / (inv_t * LOG2E);
  uint32_t bits;
  memcpy(&bits, &low, sizeof bits);
  bits &= 0xFFFF0000u;                     // towards 0
  float r;
  memcpy(&r, &bits, sizeof r);
  return r;
}

// ------------------------------------------------------------------ the largest of many keys
// Value and index of an element as one integer that grows with the value and, among equal values, with a falling index, so no two
// elements of a row have the same key and the order of ties is the order of ids.  0 is below every key.  A NaN counts as
// -inf here (its row has no numbers to report anyway); -0 and 0 are equal.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
  const float v = x == x ? x + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(v);
  const uint32_t ordered = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(ordered) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t o = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xFFFFFFFFu - static_cast<uint32_t>(k); }

// One compare-exchange step of a bitonic network over the warp: lanes `mask` apart, the larger key to the lane whose bit of
// `up` is clear.
__device__ __forceinline__ uint64_t exchange(uint64_t k, int mask, bool larger) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, k, mask);
  return (k > o) == larger ? k : o;
}

// The warp's keys, falling by lane.
__device__ __forceinline__ uint64_t sort_falling(uint64_t k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int mask = size / 2; mask > 0; mask /= 2) k = exchange(k, mask, ((lane & mask) == 0) == ((lane & size) == 0 || size == 32));
  return k;
}

// The 32 largest of two falling lists, falling: lane by lane the larger of one list and the other reversed are they, first
// rising and then falling or the other way round, which five exchanges put in order.
__device__ __forceinline__ uint64_t merge_falling(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(0xffffffffu, b, 31 - lane);
  uint64_t k = a > r ? a : r;
#pragma unroll
  for (int mask = 16; mask > 0; mask /= 2) k = exchange(k, mask, (lane & mask) == 0);
  return k;
}

// A key into a falling list, its last one out.
__device__ __forceinline__ uint64_t insert_falling(uint64_t list, uint64_t key, int lane) {
  const int at = __popc(__ballot_sync(0xffffffffu, list > key));
  const uint64_t before = __shfl_up_sync(0xffffffffu, list, 1);
  return lane < at ? list : lane == at ? key : before;
}

// The 32 largest of the lists of `n` warps (a power of two), in lists[0]; every thread of the CTA calls it with its own.
__device__ __forceinline__ void merge_lists(uint64_t own, uint64_t (*lists)[32], int n, int warp, int lane) {
  lists[warp][lane] = own;
  for (int half = n / 2; half > 0; half /= 2) {
    __syncthreads();
    if (warp < half) {
      own = merge_falling(own, lists[warp + half][lane], lane);
      lists[warp][lane] = own;
    }
  }
  __syncthreads();
}

struct Shared {
  float m[WARPS], s[WARPS], t[WARPS];
  float part_m[MAX_PARTS], part_s[MAX_PARTS], part_t[MAX_PARTS];
  uint64_t lists[WARPS][32];
  uint64_t part_lists[MAX_PARTS][32];
  uint64_t halves[2][32];
  uint64_t bound;
  int owners[THREADS], groups[THREADS];
  int num_owners, num_found;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Where a part of a row begins, how many single elements stand in front of its first 16-byte boundary, how many vectors and
// single elements follow.  Thread i takes single element i of the head and of the tail, and vectors i, i + THREADS, ...
struct Span {
  long long first;       // element of the row
  int head, vecs, tail;

  template <class T>
  __device__ __forceinline__ static Span of(const T* row, int V, int part, int parts) {
    const int len = ((V + parts - 1) / parts + 63) / 64 * 64;
    const long long lo = static_cast<long long>(part) * len, hi = min(static_cast<long long>(V), lo + len);
    const int n = hi > lo ? static_cast<int>(hi - lo) : 0;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row + lo) & 15u) / static_cast<int>(sizeof(T));
    Span s;
    s.first = lo;
    s.head = min(n, (VEC<T> - off) % VEC<T>);
    s.vecs = (n - s.head) / VEC<T>;
    s.tail = n - s.head - s.vecs * VEC<T>;
    return s;
  }
};

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A vector and the largest numbers of two halves of its elements, in the vector's own form.  bf16 elements are `low` at least, two in an
// instruction; of fp32 ones the exponents are bounded in place of that, by a constant: 4096 rows of 128256 310 us, bounded by `low`
// 328 (with alternatives, 2000 rows of 32003, 70 and 67).
template <class T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  uint4 u;
  uint32_t most;
  __device__ __forceinline__ Vec(const uint4& v, float low) {
    const uint32_t pair = __byte_perm(__float_as_uint(low), 0, 0x3232u);
    u = make_uint4(max_nan_bf16x2(v.x, pair), max_nan_bf16x2(v.y, pair), max_nan_bf16x2(v.z, pair), max_nan_bf16x2(v.w, pair));
    most = max_bf16x2(max_bf16x2(u.x, u.y), max_bf16x2(u.z, u.w));
  }
  __device__ __forceinline__ void also(const Vec& o) { most = max_bf16x2(most, o.most); }
  __device__ __forceinline__ float largest() const { return fmaxf(__uint_as_float(most << 16), __uint_as_float(most & 0xFFFF0000u)); }
  __device__ __forceinline__ void elements(float (&f)[8]) const { unpack(u, f, __nv_bfloat16()); }
};
template <>
struct Vec<float> {
  float4 u;
  float most;
  __device__ __forceinline__ Vec(const uint4& v, float) {
    u = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
    most = fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w));
  }
  __device__ __forceinline__ void also(const Vec& o) { most = fmaxf(most, o.most); }
  __device__ __forceinline__ float largest() const { return most; }
  __device__ __forceinline__ void elements(float (&f)[4]) const {
    f[0] = u.x;
    f[1] = u.y;
    f[2] = u.z;
    f[3] = u.w;
  }
};

// Sums of the quick pass: exponents are x c2 - base, one rounded operation, with the base of the largest element so far, `top`.  A
// base that stays behind it by up to 2^30, which would leave out most of the raising, costs a peaked row's entropy its last digits: terms
// of t then have both signs (error 2e-6 against 2e-7).
struct QuickSums {
  float base, top, s, t;

  __device__ __forceinline__ void raise(float x, float c2) {
    const float to = x * c2, d = max_nan(base - to, FAR_BELOW), f = ex2(d);
    t = f * fmaf(s, d, t);
    s *= f;
    base = to;
    top = x;
  }
  // ANY: x may be below low, or -inf
  template <bool ANY>
  __device__ __forceinline__ void add(float x, float c2) {
    float a = fmaf(x, c2, -base);
    if (ANY) a = max_nan(a, -200.f);                          // 2^-200 is 0 here, and so is 0 times -200
    const float w = ex2(a);
    s += w;
    t = fmaf(w, a, t);
  }
};

// Where a thread's largest element is: not in front of `first`, and not behind `last`.
struct Place {
  uint32_t first, last;
  bool any;              // the thread has elements
  int group;             // in the vectors group + j THREADS, j < AHEAD, ...
  float second;          // ... and nothing else of the thread is above this; -1: it may be anywhere
};

// A thread's sums over its elements of a span, and (TOP) where its largest is.
template <class T>
struct Pass {
  const T* row;
  const T* head;
  const T* body;
  const T* tail;
  Span sp;
  float c2, low;

  // Elements in front of and behind the vectors; `take` gets the element and its place in the row.
  template <class F>
  __device__ __forceinline__ void singles(int n, const T* from, F take) const {
    if (static_cast<int>(threadIdx.x) < n) take(to_float(from[threadIdx.x]), static_cast<uint32_t>(from - row) + threadIdx.x);
  }

  template <bool TOP>
  __device__ __forceinline__ Sums quick(Place& place) const {
    // a base that belongs to `top` as all later ones do, so that none lies below it, and far above the exponents of low
    QuickSums v = {0.5f * low * c2, 0.5f * low, 0.f, 0.f};
    float m = -INFINITY;
    float second = -INFINITY;              // what is above it is there too
    auto single = [&](float f, uint32_t at) {
      const float x = max_nan(f, low);
      if (x > m || !place.any) place = {at, at, true, -1, 0.f};
      second = fmaxf(second, fminf(x, m));
      m = fmaxf(m, x);
      if (x > v.top) v.raise(x, c2);
      v.template add<false>(x, c2);
    };
    singles(sp.head, head, single);
    int best = -1, span = 0;               // the vectors from `best`, `span` apart at most, among which the largest element is
    const uint4* vecs = reinterpret_cast<const uint4*>(body);
    int i = threadIdx.x;
    for (; i + (AHEAD - 1) * THREADS < sp.vecs; i += AHEAD * THREADS) {
      uint4 u[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) u[j] = __ldcs(vecs + i + j * THREADS);
      Vec<T> first(u[0], low), rest[AHEAD - 1] = {Vec<T>(u[1], low), Vec<T>(u[2], low), Vec<T>(u[3], low)};
      Vec<T> all = first;
#pragma unroll
      for (int j = 0; j < AHEAD - 1; ++j) all.also(rest[j]);
      const float lm = all.largest();
      if (TOP && (lm > m || !place.any)) {
        best = i;
        span = (AHEAD - 1) * THREADS;
        place.any = true;
      }
      if (TOP) second = fmaxf(second, fminf(lm, m));
      m = fmaxf(m, lm);
      if (lm > v.top) v.raise(lm, c2);
      float f[VEC<T>];
      first.elements(f);
#pragma unroll
      for (int q = 0; q < VEC<T>; ++q) v.template add<sizeof(T) == 4>(f[q], c2);
#pragma unroll
      for (int j = 0; j < AHEAD - 1; ++j) {
        rest[j].elements(f);
#pragma unroll
        for (int q = 0; q < VEC<T>; ++q) v.template add<sizeof(T) == 4>(f[q], c2);
      }
    }
#pragma unroll 1
    for (; i < sp.vecs; i += THREADS) {
      const Vec<T> x(__ldcs(vecs + i), low);
      const float lm = x.largest();
      if (TOP && (lm > m || !place.any)) {
        best = i;
        span = 0;
        place.any = true;
      }
      if (TOP) second = fmaxf(second, fminf(lm, m));
      m = fmaxf(m, lm);
      if (lm > v.top) v.raise(lm, c2);
      float f[VEC<T>];
      x.elements(f);
#pragma unroll
      for (int q = 0; q < VEC<T>; ++q) v.template add<sizeof(T) == 4>(f[q], c2);
    }
    if (TOP && best >= 0) {
      place.first = static_cast<uint32_t>(body - row) + static_cast<uint32_t>(best) * VEC<T>;
      place.last = place.first + static_cast<uint32_t>(span + 1) * VEC<T> - 1;
    }
    place.group = best;
    singles(sp.tail, tail, single);
    place.second = second;
    // of a thread with nothing above low the sums are 0, or NaN
    Sums r = {m, v.top, v.s, v.t};
    r.shift(fmaf(-r.from, c2, v.base));
    return r;
  }

  // Any numbers: element by element, from the running maximum.
  __device__ __noinline__ Sums exact(Place& place) const {
    Sums v = Sums::none();
    place.any = false;
    auto take = [&](float f, uint32_t at) {
      if (f > v.m || !place.any) place = {at, at, true, -1, 0.f};
      if (f > v.m) {
        v.rebase(fmaxf(f, -FLT_MAX), c2);
        v.m = f;
      }
      const float a = max_nan((f - v.from) * c2, FAR_BELOW), w = ex2(a);
      v.s += w;
      v.t = fmaf(w, a, v.t);
    };
    singles(sp.head, head, take);
    for (int i = threadIdx.x; i < sp.vecs; i += THREADS)
      for (int q = 0; q < VEC<T>; ++q) {
        const T* p = body + static_cast<long long>(i) * VEC<T> + q;
        take(to_float(*p), static_cast<uint32_t>(p - row));
      }
    singles(sp.tail, tail, take);
    return v;
  }
};

constexpr unsigned long long FETCH = 16384;
// The beginning of a row into L2.
template <class T>
__device__ __forceinline__ void fetch_ahead(const T* row, int V) {
  const uintptr_t first = (reinterpret_cast<uintptr_t>(row) + 15) & ~static_cast<uintptr_t>(15);
  const uintptr_t end = reinterpret_cast<uintptr_t>(row + V) & ~static_cast<uintptr_t>(15);
  if (end <= first) return;
  const uint32_t bytes = static_cast<uint32_t>(min(static_cast<unsigned long long>(end - first), FETCH));
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(first), "r"(bytes) : "memory");
}

// One CTA per row, or a cluster of `parts` CTAs where there are few rows, whose sums and lists meet in the shared memory of the
// first.  One pass over the row: every thread keeps the sums of its elements, the place of its largest and the largest outside the
// group of vectors that this is in.  For the alternatives, the threads' largest keys (taken for as small as their places allow) are
// reduced to 64, the largest of a lane number's in every other warp; the top-th largest of those is a bound that at least so many
// elements reach.  The elements that reach it belong to the few threads whose largest does, and of most of those to that one group of
// vectors, which is looked at again; what is found is sorted.  1024 rows of 128256: 50 us without alternatives, 60 with 5 or 20 (floor 40),
// of which the bound and the sorting take 2.5, looking again 4 (with all vectors of those threads 12).  Those groups kept in shared
// memory, and rows that start apart, bring nothing.
// CTAS of them share an SM, with the registers that leaves: three where there are rows for them, so that others read while one
// looks for its alternatives (2048 x 128256 with 20: 127 us by two, 110 by three); two, each of them faster, where there are not (296 rows
// 22 and 28 us).  Without alternatives three are as fast with few rows.
// The row that a later CTA is likely to take next here, `later` rows on, is fetched in part while the warps wait for one another: 1024
// rows without alternatives 56 -> 50 us, 4096 rows 171-183 -> 172 (floor 160); with alternatives no gain, and none taken.
template <class T, bool TOP, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS)
logprobs_fwd_kernel(const T* __restrict__ logits, const long long* __restrict__ tokens, float* __restrict__ logprob,
                    float* __restrict__ entropy, float* __restrict__ top_logprob, long long* __restrict__ top_id,
                    float* __restrict__ stats, int V, long long ld, long long ignore_index, int top, int parts, float inv_t, float low,
                    long long later) {
  if (parts > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  grid_begin(logits, tokens);
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - row * parts);
  const T* x = logits + row * ld;
  const Span sp = Span::of(x, V, part, parts);
  const T* head = x + sp.first;
  const T* body = head + sp.head;
  const T* tail = body + static_cast<long long>(sp.vecs) * VEC<T>;
  const float c2 = inv_t * LOG2E;
  const Pass<T> pass = {x, head, body, tail, sp, c2, low};

  Sums v;
  uint64_t bound = 0;
  Place place = {0, 0, false, -1, 0.f};
  for (int exact = 0; exact < 2; ++exact) {
    v = exact ? pass.exact(place) : pass.template quick<TOP>(place);
    if (!TOP && parts == 1 && threadIdx.x == 0 && exact == 0 && row + later < gridDim.x) fetch_ahead(x + later * ld, V);
    const float wm = warp_max(v.m);
    if (lane == 0) sh.m[warp] = wm;
    if (TOP) sh.lists[warp][lane] = place.any ? make_key(v.m, place.last) : 0;
    __syncthreads();
    if (TOP && warp < 2) {
      uint64_t k = sh.lists[warp][lane];
#pragma unroll
      for (int w = 2; w < WARPS; w += 2) k = max(k, sh.lists[warp + w][lane]);
      k = sort_falling(k, lane);
      sh.halves[warp][lane] = k;
      asm volatile("bar.sync 1, 64;" ::: "memory");
      if (warp == 0) {
        k = merge_falling(k, sh.halves[1][lane], lane);
        if (lane == top - 1) sh.bound = k;
        if (lane == 0) sh.num_owners = sh.num_found = 0;
      }
    }
    const uint64_t most = TOP && place.any ? make_key(v.m, place.first) : 0;
    v.m = sh.m[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v.m = fmaxf(v.m, sh.m[w]);
    __syncthreads();
    bool good = fabsf(v.m) < -0.5f * low;
    if (TOP) {
      bound = sh.bound;
      good = good && (bound == 0 || key_value(bound) > low);
      if ((good || exact) && most != 0 && most >= bound) {
        const int at = atomicAdd(&sh.num_owners, 1);
        sh.owners[at] = threadIdx.x;
        sh.groups[at] = bound != 0 && place.second < key_value(bound) ? place.group : -1;
      }
    }
    if (good || exact) break;
    __syncthreads();                       // read before it is written again
  }
  v.rebase(fmaxf(v.m, -FLT_MAX), c2);
  const float ws = warp_sum(v.s), wt = warp_sum(v.t);
  if (lane == 0) {
    sh.s[warp] = ws;
    sh.t[warp] = wt;
  }
  __syncthreads();

  uint64_t list = 0;
  if (TOP) {
    // A found key into the buffer that the lists were in; there is room for THREADS.
    uint64_t* const found = &sh.lists[0][0];
    auto offer = [&](float f, uint32_t index) {
      const uint64_t key = make_key(f, index);
      if (key >= bound) {
        const int at = atomicAdd(&sh.num_found, 1);
        if (at < THREADS) found[at] = key;
      }
    };
    const float least = bound == 0 ? -INFINITY : key_value(bound);
    auto offer_vec = [&](int at) {
      const uint4 u = reinterpret_cast<const uint4*>(body)[at];
      // most vectors have nothing that reaches the bound; NaN counts as -inf, which reaches it if it is as low
      if (Vec<T>(u, low).largest() < least) return;
      float f[VEC<T>];
      unpack(u, f, T());
      const uint32_t first = static_cast<uint32_t>(body - x) + static_cast<uint32_t>(at) * VEC<T>;
#pragma unroll
      for (int q = 0; q < VEC<T>; ++q) offer(f[q], first + q);
    };
    // Of most owners only the group of vectors that their largest element is in, a vector per thread; of the others all vectors,
    // lane by lane.
    const int owners = sh.num_owners;
    for (int i = threadIdx.x; i < owners * AHEAD; i += THREADS) {
      const int group = sh.groups[i / AHEAD], at = group + i % AHEAD * THREADS;
      if (group >= 0 && at < sp.vecs) offer_vec(at);
    }
    for (int o = warp; o < owners; o += WARPS)
      if (sh.groups[o] < 0)
        for (int at = sh.owners[o] + lane * THREADS; at < sp.vecs; at += 32 * THREADS) offer_vec(at);
    for (int e = threadIdx.x; e < owners; e += THREADS) {
      const int owner = sh.owners[e];
      if (owner < sp.head) offer(to_float(head[owner]), static_cast<uint32_t>(head + owner - x));
      if (owner < sp.tail) offer(to_float(tail[owner]), static_cast<uint32_t>(tail + owner - x));
    }
    __syncthreads();
    const int n = sh.num_found;
    if (n <= THREADS) {
      if (warp == 0 || n > 32) list = sort_falling(static_cast<int>(threadIdx.x) < n ? found[threadIdx.x] : 0, lane);
      if (n > 32) {
        __syncthreads();
        merge_lists(list, sh.lists, WARPS, warp, lane);
        list = sh.lists[0][lane];
      }
    } else {
      // rows of many equal logits: every warp puts what it finds into a list of its own
      __syncthreads();
      auto insert = [&](bool has, float f, uint32_t index) {
        const uint64_t key = has ? make_key(f, index) : 0;
        const uint64_t least = __shfl_sync(0xffffffffu, list, 31);       // by all lanes, in front of any condition
        unsigned waiting = __ballot_sync(0xffffffffu, key >= bound && key > least);
        while (waiting != 0) {
          const int from = __ffs(waiting) - 1;
          waiting &= waiting - 1;
          list = insert_falling(list, __shfl_sync(0xffffffffu, key, from), lane);
        }
      };
      list = 0;
      for (int e = warp; e < owners; e += WARPS) {
        const int owner = sh.owners[e];
        const bool at_head = lane == 0 && owner < sp.head, at_tail = lane == 1 && owner < sp.tail;
        const T* s = at_head ? head + owner : tail + owner;
        insert(at_head || at_tail, at_head || at_tail ? to_float(*s) : 0.f, static_cast<uint32_t>(s - x));
        for (int i0 = owner; i0 < sp.vecs; i0 += 32 * THREADS) {
          const int i = i0 + lane * THREADS;
          const bool has = i < sp.vecs;
          float f[VEC<T>];
          unpack(has ? reinterpret_cast<const uint4*>(body)[i] : make_uint4(0, 0, 0, 0), f, T());
          const uint32_t at = static_cast<uint32_t>(body - x) + static_cast<uint32_t>(i) * VEC<T>;
#pragma unroll
          for (int q = 0; q < VEC<T>; ++q) insert(has, f[q], at + q);
        }
      }
      merge_lists(list, sh.lists, WARPS, warp, lane);
      list = sh.lists[0][lane];
    }
  }
  if (warp == 0) {
    v.s = warp_sum(lane < WARPS ? sh.s[lane] : 0.f);
    v.t = warp_sum(lane < WARPS ? sh.t[lane] : 0.f);
  }
  if (parts > 1) {
    // the sums and the list of every part into the first CTA of the cluster, which has started by now
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 0) {
      auto put = [](float* at, float f) {
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_u32(smem_u32(at), 0)), "f"(f) : "memory");
      };
      if (lane == 0) {
        put(&sh.part_m[part], v.m);
        put(&sh.part_s[part], v.s);
        put(&sh.part_t[part], v.t);
      }
      if (TOP)
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(mapa_u32(smem_u32(&sh.part_lists[part][lane]), 0)), "l"(list)
                     : "memory");
    }
    cluster_sync();
    if (part != 0 || warp != 0) return;
    v = Sums::none();
    if (lane < parts) {
      v.m = sh.part_m[lane];
      v.from = fmaxf(v.m, -FLT_MAX);
      v.s = sh.part_s[lane];
      v.t = sh.part_t[lane];
    }
    v.m = warp_max(v.m);
    v.rebase(fmaxf(v.m, -FLT_MAX), c2);
    v.s = warp_sum(v.s);
    v.t = warp_sum(v.t);
    if (TOP)
      for (int p = 1; p < parts; ++p) list = merge_falling(list, sh.part_lists[p][lane], lane);
  } else if (warp != 0) {
    return;
  }
  const bool empty = v.s == 0.f;           // nothing left: every probability is 0
  const float log_s = empty ? -INFINITY : log2f(v.s);
  auto log_p = [&](float f) { return empty ? -INFINITY : fmaf(f - v.from, inv_t, -log_s * LN2); };
  if (lane == 0) {
    const long long y = tokens[row];
    const bool counted = y != ignore_index && y >= 0 && y < V;
    logprob[row] = counted ? log_p(to_float(x[y])) : 0.f;
    entropy[row] = empty ? 0.f : (log_s - v.t / v.s) * LN2;
    stats[2 * row] = v.from;
    stats[2 * row + 1] = log_s;
  }
  if (TOP && lane < top) {
    top_logprob[row * top + lane] = log_p(key_value(list));
    top_id[row * top + lane] = key_index(list);
  }
}

// dx of one part of a row by one CTA, then the elements of the token and of the alternatives again with their g.  One read and one write
// of the logits bound it: 4096 rows of 128256 in bf16 337 us (floor 321), the forward pass without alternatives 172 (160).
template <class T, bool ALIGNED>
__global__ void __launch_bounds__(THREADS, 2)
logprobs_bwd_kernel(const T* __restrict__ logits, const long long* __restrict__ tokens, const float* __restrict__ stats,
                    const float* __restrict__ entropy, const long long* __restrict__ top_id,
                    const float* __restrict__ d_logprob, const float* __restrict__ d_entropy, const float* __restrict__ d_top,
                    T* __restrict__ d, int V, long long ld, long long ignore_index, int top, int parts, float inv_t) {
  grid_begin(logits, tokens, stats, entropy, top_id, d_logprob, d_entropy, d_top);
  const long long row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x - row * parts);
  const T* x = logits + row * ld;
  T* o = d + row * V;
  const Span sp = Span::of(x, V, part, parts);
  const long long y = tokens[row];
  const bool counted = y != ignore_index && y >= 0 && y < V;
  const float from = stats[2 * row], log_s = stats[2 * row + 1], h = entropy[row];
  const float gy = counted && d_logprob != nullptr ? d_logprob[row] : 0.f;
  const float gh = d_entropy != nullptr ? d_entropy[row] : 0.f;
  float g = gy;
  bool live = gy != 0.f || gh != 0.f;
  if (d_top != nullptr)
    for (int i = 0; i < top; ++i) {
      g += d_top[row * top + i];
      live = live || d_top[row * top + i] != 0.f;
    }
  if (!live || log_s == -INFINITY) {
    // nothing asks for this row (padding, whatever its logits are), or nothing is left in it: its logits are not read
    const Span out = Span::of(o, V, part, parts);
    T* const first = o + out.first;
    const int t = threadIdx.x;
    if (t < out.head) from_float(0.f, first[t]);
    if (t < out.tail) from_float(0.f, first[out.head + static_cast<long long>(out.vecs) * VEC<T> + t]);
    for (int i = t; i < out.vecs; i += THREADS) reinterpret_cast<uint4*>(first + out.head)[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  // dx = 2^u (a + b u) with u = log2 p
  const float c2 = inv_t * LOG2E;
  const float a = -(g + gh * h) * inv_t, b = -gh * LN2 * inv_t;
  auto grad = [&](float f) {
    const float u = max_nan(fmaf(f - from, c2, -log_s), -200.f);      // 2^-200 is 0 here, and so is 0 (a - 200 b)
    return ex2(u) * fmaf(b, u, a);
  };
  const long long begin = sp.first, end = begin + sp.head + static_cast<long long>(sp.vecs) * VEC<T> + sp.tail;
  if (ALIGNED) {                       // x and o have the same offset to a 16-byte boundary
    const long long body = begin + sp.head, tail = end - sp.tail;
    const int t = threadIdx.x;
    if (t < sp.head) from_float(grad(to_float(x[begin + t])), o[begin + t]);
    if (t < sp.tail) from_float(grad(to_float(x[tail + t])), o[tail + t]);
    for (int i = t; i < sp.vecs; i += AHEAD * THREADS) {
      uint4 u[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (i + j * THREADS < sp.vecs) u[j] = __ldcs(reinterpret_cast<const uint4*>(x + body) + i + j * THREADS);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (i + j * THREADS >= sp.vecs) break;
        float f[VEC<T>];
        unpack(u[j], f, T());
#pragma unroll
        for (int q = 0; q < VEC<T>; ++q) f[q] = grad(f[q]);
        reinterpret_cast<uint4*>(o + body)[i + j * THREADS] = pack(f, T());
      }
    }
  } else {
    for (long long i = begin + threadIdx.x; i < end; i += THREADS) from_float(grad(to_float(x[i])), o[i]);
  }
  __syncthreads();
  // the token may be one of the alternatives: whoever writes a place has all that belongs to it
  const int who = static_cast<int>(threadIdx.x);
  const int listed = d_top != nullptr ? top : 0;
  if (who > listed || (who == listed && !counted)) return;
  auto id = [&](int i) { return i < listed ? top_id[row * top + i] : y; };
  const long long at = id(who);
  if (at < begin || at >= end) return;
  float sum = 0.f;
  for (int i = 0; i <= listed; ++i)
    if (i < listed ? id(i) == at : counted && y == at) sum += i < listed ? d_top[row * top + i] : gy;
  from_float(fmaf(sum, inv_t, grad(to_float(x[at]))), o[at]);
}

// CTAs per row: with fewer rows than SMs have room for, a row is cut into up to eight pieces of at least 4,096 elements.  Not with
// more rows, where a cluster waits for SMs together: 296 rows of 128256 with 20 alternatives 22.5 us, in four pieces 42; 1024 rows 60 us,
// in two 83, without alternatives 50 and 65.  One row of 128256 5.2 us, in one piece 8.7.  For rows of a quarter of that the forward pass
// loses by it what waiting for the cluster costs: 37 rows of 32003 6.8 us, in one piece 5.4 (with 20 alternatives 9.4 and 7.9; of fp32
// without alternatives 7.0 and 8.1), 74 rows 7.9 and 6.4 (14.8 and 8.5), one row 4.6 either way; and where eight pieces fill the
// SMs, alternatives do: 37 rows of 128256 17.7, in four 12.8, without alternatives 9.5 and 10.5.  The backward pass, whose pieces need no
// cluster, gains: 37 rows of 32003 3.0 us, in one piece 4.6; 37 of 128256 4.7 and 11.9.
int row_parts(long long T, int V, int num_sms) {
  int parts = 1;
  while (parts < MAX_PARTS && T * parts * 2 <= 2ll * num_sms && V / (parts * 2) >= 4096) parts *= 2;
  return parts;
}

template <class... P, class... A>
int launch_clusters(void (*kernel)(P...), long long grid, int cluster, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) == cudaSuccess ? 0 : -3;
}

template <class T>
int fwd(const LogprobArgs& a, float* logprob, float* entropy, float* top_logprob, long long* top_id, float* stats, int num_sms,
        cudaStream_t st) {
  const int parts = row_parts(a.T, a.V, num_sms);
  auto kernel = a.top == 0                    ? logprobs_fwd_kernel<T, false, 3>
                : a.T * parts > 2ll * num_sms ? logprobs_fwd_kernel<T, true, 3>
                                              : logprobs_fwd_kernel<T, true, 2>;
  const bool three = a.top == 0 || a.T * parts > 2ll * num_sms;
  const long long later = (three ? 3ll : 2ll) * num_sms;
  return launch_clusters(kernel, a.T * parts, parts, st, static_cast<const T*>(a.logits), a.tokens, logprob, entropy, top_logprob,
                         top_id, stats, a.V, a.ld, a.ignore_index, a.top, parts, a.inv_temperature, lowest_logit(a.inv_temperature),
                         later);
}

template <class T>
int bwd(const LogprobArgs& a, const float* stats, const float* entropy, const long long* top_id, const float* d_logprob,
        const float* d_entropy, const float* d_top, void* d, int num_sms, cudaStream_t st) {
  const int parts = row_parts(a.T, a.V, num_sms);
  const uintptr_t apart = reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(d);
  const bool aligned = (apart & 15u) == 0 && (a.T <= 1 || (a.ld - a.V) * sizeof(T) % 16 == 0);
  auto kernel = aligned ? logprobs_bwd_kernel<T, true> : logprobs_bwd_kernel<T, false>;
  return launch_clusters(kernel, a.T * parts, 1, st, static_cast<const T*>(a.logits), a.tokens, stats, entropy, top_id, d_logprob,
                         d_entropy, d_top, static_cast<T*>(d), a.V, a.ld, a.ignore_index, a.top, parts, a.inv_temperature);
}

bool sound(const LogprobArgs& a) {
  return a.T >= 0 && a.T <= (1ll << 27) && a.V > 0 && a.V <= kMaxVocabulary && a.top >= 0 && a.top <= kMaxTopTokens && a.top <= a.V;
}

}  // namespace

int logprobs_fwd(const LogprobArgs& a, float* logprob, float* entropy, float* top_logprob, long long* top_id, float* stats,
                 int num_sms, cudaStream_t st) {
  if (!sound(a)) return -1;
  if (a.T == 0) return 0;
  return a.f32 ? fwd<float>(a, logprob, entropy, top_logprob, top_id, stats, num_sms, st)
               : fwd<__nv_bfloat16>(a, logprob, entropy, top_logprob, top_id, stats, num_sms, st);
}

int logprobs_bwd(const LogprobArgs& a, const float* stats, const float* entropy, const long long* top_id,
                 const float* d_logprob, const float* d_entropy, const float* d_top, void* d, int num_sms, cudaStream_t st) {
  if (!sound(a)) return -1;
  if (a.T == 0) return 0;
  return a.f32 ? bwd<float>(a, stats, entropy, top_id, d_logprob, d_entropy, d_top, d, num_sms, st)
               : bwd<__nv_bfloat16>(a, stats, entropy, top_id, d_logprob, d_entropy, d_top, d, num_sms, st);
}

}  // namespace piper
