// One AdamW step over many tensors in one launch, moments held in 32 or in 8 bits:
//
//   g = grad * grad_scale,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// What bounds it: memory.  An element moves 4 (or 2) bytes of gradient, 8 of weight, 2 of a bf16 parameter, and 16 of moments in 32
// bits, 4 in 8 bits (and a scale of 4 bytes for 256 elements, in and out).
//
// 8-bit moments.  A block of 256 elements keeps its largest magnitude as its scale, in fp32 and without rounding, so that
// what all of a block has in common (the decay of v under small gradients above all) is not rounded at all.  The rest, y = |x| / scale in [0, 1],
// keeps the upper bits of its fp32 form: three bits of mantissa, and as many binades below 1 as there are codes for, 16 for m beside its
// sign, 32 for v; code 0 is 0.  Rounding is up or down in proportion to the distance: v moves by (1 - b2) of
// itself in a step, far less than half the distance of two codes, and rounded to the nearest it would never move; this way it
// moves on average as it should.  A v above 0 never becomes 0, which would make its weight's step unbounded.  The random bits
// come from the step, the tensor's place in the list and the element's index, so a step from the same state has the same bits.
// All operations up to the code are single, rounded fp32 operations in a fixed order (no fused multiply-add): codes are the
// same wherever the definition is followed.
#include "adamw.h"

#include <cuda_bf16.h>

#include <cstdint>

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CHUNK_BLOCKS = WARPS;                      // blocks of a chunk, one per warp
constexpr int CHUNK = CHUNK_BLOCKS * kMomentBlock;
constexpr int PER = kMomentBlock / 32;                   // elements of a lane
constexpr int M_BASE = 889, V_BASE = 761;                // fp32 bits >> 20 of code 0: those of 1.0 are 1016, codes 127 and 255

// Code in byte `Byte` of a word to its value.  A byte moved to bits 16-23 is a multiplication away from the upper bits of the number.
template <int BYTE>
__device__ __forceinline__ float decode_v(uint32_t word, float scale) {
  const uint32_t c = __byte_perm(word, 0, 0x4044u | BYTE << 8);
  return __fmul_rn(__uint_as_float(c != 0 ? c * 16 + (static_cast<uint32_t>(V_BASE) << 20) : 0u), scale);
}
template <int BYTE>
__device__ __forceinline__ float decode_m(uint32_t word, float scale) {
  const uint32_t c = __byte_perm(word, 0, 0x4044u | BYTE << 8), low = c & 0x7F0000u;
  const uint32_t bits = low != 0 ? low * 16 + (static_cast<uint32_t>(M_BASE) << 20) : 0u;
  return __fmul_rn(__uint_as_float(bits | (c << 8 & 0x80000000u)), scale);
}

// Codes of y in [0, 1], in the top byte of the result: the upper bits of y plus what 16 random bits (the lower or the upper ones of r)
// carry into them; below code 1, 0 or 1 (v: 1 for all that is above 0).  Bits 20-27 of y and the base are brought to the top
// byte by a shift, whose overflow is what the base takes away.
constexpr uint32_t M_LEAST = static_cast<uint32_t>(M_BASE + 1) << 20, V_LEAST = static_cast<uint32_t>(V_BASE + 1) << 20;
__device__ __forceinline__ uint32_t encode_m(float y, uint32_t r) {
  return (__float_as_uint(y) << 4) + __byte_perm(r, (256u - M_BASE % 256) << 24, 0x7104u);
}
__device__ __forceinline__ uint32_t encode_v(float y, uint32_t r) {
  return (__float_as_uint(y) << 4) + __byte_perm(r, (256u - V_BASE % 256) << 24, 0x7324u);
}
__device__ __forceinline__ uint32_t encode_small_m(float y, uint32_t r) {
  return __fmul_rn(static_cast<float>(r & 0xFFFFu), __uint_as_float(M_LEAST) * (1.f / 65536)) < y ? 1u << 24 : 0u;
}
__device__ __forceinline__ uint32_t encode_small_v(float v) { return v > 0.f ? 1u << 24 : 0u; }

// The top bytes of four words, the first lowest.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&t)[4]) {
  return __byte_perm(__byte_perm(t[0], t[1], 0x0073u), __byte_perm(t[2], t[3], 0x0073u), 0x5410u);
}

// The block's largest magnitude, NaN where a value is infinite or NaN.
__device__ __forceinline__ float block_scale(const float (&x)[PER]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(x[i])));
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7FFFFFFFu);
  return bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(bits);
}

// The rare operations, out of the way of the common ones in the instruction cache.
__device__ __noinline__ float divide(float a, float b) { return __fdiv_rn(a, b); }
__device__ __noinline__ float small_eps_update(float m, float v, float root, float eps) {
  if (eps < 1e-30f) return m / fmaf(sqrtf(v), root, eps);
  float r, q;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  asm("div.approx.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(fmaf(r, root, eps)));
  return q;
}

// y = |x| / scale of a block, correctly rounded.  With the correctly rounded reciprocal, a product, its exact remainder and a
// correction give the quotient (Markstein, IBM J. Res. Dev. 34, 1990) where nothing underflows: a quotient that is not small enough for
// code 0 or 1 anyway comes from x above 2^-101, whose remainder is a normal number, if the scale is above 2^-60.  Other blocks
// divide.
__device__ __forceinline__ void quotients(const float* x, float scale, float (&y)[4]) {
  const float s = scale > 0.f ? scale : 1.f;
  if (s >= 8.67361738e-19f && s <= 1.f) {
    const float inverse = __frcp_rn(s);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = fabsf(x[j]), q = __fmul_rn(a, inverse);
      y[j] = __fmaf_rn(__fmaf_rn(-q, s, a), inverse, q);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = divide(fabsf(x[j]), s);
  }
}

// m / (sqrt(v) root + eps), within two units of the last place for the root and for the quotient.  Where eps is small enough for the
// root of a v below the normal numbers to matter beside it (`small_eps`), that is not taken for 0: 64 Mi elements with 8-bit
// moments 257 us in place of 222; within the common path that is 241, but 224 for all others.  A vanishing eps, beside which a denominator
// may be below them, takes the exact operations.
__device__ __forceinline__ float update(float m, float v, float root, float eps, int small_eps) {
  if (small_eps) return small_eps_update(m, v, root, eps);
  float r, q;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(q) : "f"(m), "f"(fmaf(r, root, eps)));
  return q;
}

__device__ __forceinline__ void load4(const float* p, float (&x)[PER], int h) {
  const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
  x[4 * h] = v.x;
  x[4 * h + 1] = v.y;
  x[4 * h + 2] = v.z;
  x[4 * h + 3] = v.w;
}
__device__ __forceinline__ void store4(float* p, const float (&x)[PER], int h) {
  *reinterpret_cast<float4*>(p) = make_float4(x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]);
}

// A warp takes a block: lane l has elements 4 l to 4 l + 3 of either half, so that its vectors are neighbours of the next lane's.
// The CTAs that are resident walk the chunks together, a block per warp at a time: 64 Mi elements with 8-bit moments and bf16
// parameters 222 us (floor 184), with 16 blocks per chunk 249 us, with twice the CTAs 267; 32-bit moments and bf16
// gradients 294 us (287), with three CTAs per SM 330 us.  Without the 8-bit arithmetic the same accesses take 212 us.  Blocks fetched two ahead through shared
// memory bring nothing (268 us in either form, with chunks of 16).
template <int BITS>
constexpr int CTAS = BITS == 8 ? 4 : 2;
template <int BITS>
__global__ void __launch_bounds__(THREADS, CTAS<BITS>)
adamw_kernel(const __grid_constant__ AdamwTable table, const AdamwArgs a) {
  grid_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = table.first[table.count];
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    int lo = 0, hi = table.count - 1;                    // the tensor of the chunk
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (table.first[mid] <= chunk) lo = mid;
      else hi = mid - 1;
    }
    const AdamwTensor& t = table.t[lo];
    const long long n = t.n;
    const float rate = t.rate, root = t.root;
    const bool aligned = ((reinterpret_cast<uintptr_t>(t.weight) | reinterpret_cast<uintptr_t>(t.grad) |
                           reinterpret_cast<uintptr_t>(t.param)) & 15u) == 0;
    {
      const long long i0 = (static_cast<long long>(chunk - table.first[lo]) * CHUNK_BLOCKS + warp) * kMomentBlock;
      if (i0 >= n) continue;
      const bool whole = i0 + kMomentBlock <= n, vec = whole && aligned;
      const long long i = i0 + lane * 4, s = t.at + i, block = (t.at + i0) / kMomentBlock;
      // element of register j, and whether it exists
      auto at = [&](int j) { return i + (j / 4) * 128 + (j & 3); };
      auto is = [&](int j) { return whole || at(j) < n; };
      float w[PER], g[PER], m[PER], v[PER];
      uint32_t mc[2], vc[2];
      float ms = 0.f, vs = 0.f;
      if (BITS == 8) {
        // the moments' buffers are aligned and hold whole blocks, zeros behind the end
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.m) + s + 128 * h);
          vc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + s + 128 * h);
        }
        ms = a.m_scale[block];
        vs = a.v_scale[block];
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load4(static_cast<const float*>(a.m) + s + 128 * h, m, h);
          load4(static_cast<const float*>(a.v) + s + 128 * h, v, h);
        }
      }
      if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h) load4(t.weight + i + 128 * h, w, h);
        if (t.grad_bf16) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint2 u = __ldcs(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(t.grad) + i + 128 * h));
            g[4 * h] = __uint_as_float(u.x << 16);
            g[4 * h + 1] = __uint_as_float(u.x & 0xFFFF0000u);
            g[4 * h + 2] = __uint_as_float(u.y << 16);
            g[4 * h + 3] = __uint_as_float(u.y & 0xFFFF0000u);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) load4(static_cast<const float*>(t.grad) + i + 128 * h, g, h);
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          w[j] = is(j) ? t.weight[at(j)] : 0.f;
          g[j] = !is(j) ? 0.f
                 : t.grad_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(t.grad)[at(j)])
                               : static_cast<const float*>(t.grad)[at(j)];
        }
      }
      if (BITS == 8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          m[4 * h] = decode_m<0>(mc[h], ms);
          m[4 * h + 1] = decode_m<1>(mc[h], ms);
          m[4 * h + 2] = decode_m<2>(mc[h], ms);
          m[4 * h + 3] = decode_m<3>(mc[h], ms);
          v[4 * h] = decode_v<0>(vc[h], vs);
          v[4 * h + 1] = decode_v<1>(vc[h], vs);
          v[4 * h + 2] = decode_v<2>(vc[h], vs);
          v[4 * h + 3] = decode_v<3>(vc[h], vs);
        }
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float gj = __fmul_rn(g[j], a.grad_scale);
        m[j] = __fadd_rn(__fmul_rn(m[j], a.b1), __fmul_rn(gj, a.c1));
        v[j] = __fadd_rn(__fmul_rn(v[j], a.b2), __fmul_rn(__fmul_rn(gj, a.c2), gj));
        w[j] = fmaf(-rate, update(m[j], v[j], root, a.eps, a.small_eps), w[j] * a.keep);
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (!is(j)) m[j] = v[j] = 0.f;
      }
      if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          store4(t.weight + i + 128 * h, w, h);
          if (t.param != nullptr)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(t.param) + i + 128 * h) =
                make_uint2(pack_bf16x2(w[4 * h], w[4 * h + 1]), pack_bf16x2(w[4 * h + 2], w[4 * h + 3]));
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (is(j)) {
            t.weight[at(j)] = w[j];
            if (t.param != nullptr) static_cast<__nv_bfloat16*>(t.param)[at(j)] = __float2bfloat16(w[j]);
          }
        }
      }
      if (BITS == 8) {
        ms = block_scale(m);
        vs = block_scale(v);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float ym[4], yv[4];
          quotients(m + 4 * h, ms, ym);
          quotients(v + 4 * h, vs, yv);
          uint32_t cm[4], cv[4], least_m = 0xFFFFFFFFu, least_v = 0xFFFFFFFFu;
          const uint32_t first = static_cast<uint32_t>(at(4 * h)) + t.seed;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t r = mix32(first + j);
            cm[j] = encode_m(ym[j], r);
            cv[j] = encode_v(yv[j], r);
            least_m = min(least_m, __float_as_uint(ym[j]));
            least_v = min(least_v, __float_as_uint(yv[j]));
          }
          if (__builtin_expect(least_m < M_LEAST || least_v < V_LEAST, 0)) {      // few have such small elements, or zeros
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (__float_as_uint(ym[j]) < M_LEAST) cm[j] = encode_small_m(ym[j], mix32(first + j));
              if (__float_as_uint(yv[j]) < V_LEAST) cv[j] = encode_small_v(v[4 * h + j]);      // y may be below all numbers
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) cm[j] = (cm[j] & 0x7FFFFFFFu) | (__float_as_uint(m[4 * h + j]) & 0x80000000u);
          mc[h] = top_bytes(cm);
          vc[h] = top_bytes(cv);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __stcs(reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.m) + s + 128 * h), mc[h]);
          __stcs(reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.v) + s + 128 * h), vc[h]);
        }
        if (lane == 0) {
          a.m_scale[block] = ms;
          a.v_scale[block] = vs;
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          store4(static_cast<float*>(a.m) + s + 128 * h, m, h);
          store4(static_cast<float*>(a.v) + s + 128 * h, v, h);
        }
      }
    }
  }
}

constexpr int DECODE_AHEAD = 4;

// Both moments: a thread has four codes of each in `AHEAD` places, all loaded before the first is written.  Memory bounds it, four
// fifths of it writes: 200 Mi elements 327 us (floor 320); by resident CTAs that walk the codes 400.
__global__ void __launch_bounds__(256)
moments_decode_kernel(const uint32_t* __restrict__ m, const float* __restrict__ m_scale, const uint32_t* __restrict__ v,
                      const float* __restrict__ v_scale, float4* __restrict__ out_m, float4* __restrict__ out_v, long long words) {
  grid_begin(m, m_scale, v, v_scale);
  constexpr int AHEAD = DECODE_AHEAD;
  {
    const long long i = static_cast<long long>(blockIdx.x) * 256 * AHEAD + threadIdx.x;
    uint32_t cm[AHEAD], cv[AHEAD];
    float sm[AHEAD], sv[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const long long at = i + 256 * k;
      if (at >= words) break;
      cm[k] = __ldcs(m + at);
      cv[k] = __ldcs(v + at);
      sm[k] = m_scale[at / (kMomentBlock / 4)];
      sv[k] = v_scale[at / (kMomentBlock / 4)];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const long long at = i + 256 * k;
      if (at >= words) break;
      __stcs(out_m + at, make_float4(decode_m<0>(cm[k], sm[k]), decode_m<1>(cm[k], sm[k]), decode_m<2>(cm[k], sm[k]),
                                     decode_m<3>(cm[k], sm[k])));
      __stcs(out_v + at, make_float4(decode_v<0>(cv[k], sv[k]), decode_v<1>(cv[k], sv[k]), decode_v<2>(cv[k], sv[k]),
                                     decode_v<3>(cv[k], sv[k])));
    }
  }
}

}  // namespace

int adamw_launch(AdamwTable& table, AdamwArgs a, int num_sms, cudaStream_t st) {
  long long chunks = 0;
  a.small_eps = 0;
  for (int i = 0; i < table.count; ++i) {
    // 2^-63, the root of the smallest normal number, times root: 2^-22 of eps or more
    if (a.eps < 4.5474735e-13f * table.t[i].root) a.small_eps = 1;
    table.first[i] = static_cast<int>(chunks);
    chunks += (table.t[i].n + CHUNK - 1) / CHUNK;
    if (chunks > INT32_MAX / 2) return -1;
  }
  table.first[table.count] = static_cast<int>(chunks);
  if (chunks == 0) return 0;
  const long long most = static_cast<long long>(a.m_scale != nullptr ? CTAS<8> : CTAS<32>) * num_sms;
  const dim3 grid(static_cast<unsigned>(chunks < most ? chunks : most));
  const cudaError_t e = a.m_scale != nullptr ? launch_overlapped(adamw_kernel<8>, grid, THREADS, 0, st, table, a)
                                             : launch_overlapped(adamw_kernel<32>, grid, THREADS, 0, st, table, a);
  return e == cudaSuccess ? 0 : -3;
}

int moments_decode(const void* m, const float* m_scale, const void* v, const float* v_scale, float* out_m, float* out_v, long long n,
                   cudaStream_t st) {
  if (n == 0) return 0;
  const long long ctas = (n / 4 + 256 * DECODE_AHEAD - 1) / (256 * DECODE_AHEAD);
  if (ctas > INT32_MAX) return -1;
  const dim3 grid(static_cast<unsigned>(ctas));
  return launch_overlapped(moments_decode_kernel, grid, 256, 0, st, static_cast<const uint32_t*>(m), m_scale,
                           static_cast<const uint32_t*>(v), v_scale, reinterpret_cast<float4*>(out_m),
                           reinterpret_cast<float4*>(out_v), n / 4) == cudaSuccess ? 0 : -3;
}

}  // namespace piper
