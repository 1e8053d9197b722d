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
constexpr int CHUNK_BLOCKS = 16;                         // blocks of a chunk, two per warp
constexpr int CHUNK = CHUNK_BLOCKS * kMomentBlock;
constexpr int PER = kMomentBlock / 32;                   // elements of a lane
constexpr int M_BASE = 889, V_BASE = 761;                // fp32 bits >> 20 of code 0: those of 1.0 are 1016, codes 127 and 255

__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

__device__ __forceinline__ float decode_v(uint32_t c, float scale) {
  return __fmul_rn(c != 0 ? __uint_as_float((c + V_BASE) << 20) : 0.f, scale);
}
__device__ __forceinline__ float decode_m(uint32_t c, float scale) {
  const uint32_t low = c & 127u;
  const float x = __fmul_rn(low != 0 ? __uint_as_float((low + M_BASE) << 20) : 0.f, scale);
  return c >= 128u ? -x : x;
}

// y in [0, 1] to its code; r: 16 random bits.
__device__ __forceinline__ uint32_t encode_m(float y, uint32_t r) {
  constexpr uint32_t least = static_cast<uint32_t>(M_BASE + 1) << 20;
  if (__float_as_uint(y) < least)
    return __fmul_rn(static_cast<float>(r), __uint_as_float(least) * (1.f / 65536)) < y ? 1u : 0u;
  return ((__float_as_uint(y) + (r << 4)) >> 20) - M_BASE;
}
__device__ __forceinline__ uint32_t encode_v(float y, uint32_t r) {
  constexpr uint32_t least = static_cast<uint32_t>(V_BASE + 1) << 20;
  if (__float_as_uint(y) < least) return y > 0.f ? 1u : 0u;
  return ((__float_as_uint(y) + (r << 4)) >> 20) - V_BASE;
}

// The block's largest magnitude, NaN where a value is infinite or NaN.
__device__ __forceinline__ float block_scale(const float (&x)[PER]) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  most = __reduce_max_sync(0xffffffffu, most);
  return most >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(most);
}

template <int BITS>
__global__ void __launch_bounds__(THREADS)
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
    const uintptr_t low = reinterpret_cast<uintptr_t>(t.weight) | reinterpret_cast<uintptr_t>(t.grad) |
                          reinterpret_cast<uintptr_t>(t.param);
    for (int b = warp; b < CHUNK_BLOCKS; b += WARPS) {
      const long long i0 = (static_cast<long long>(chunk - table.first[lo]) * CHUNK_BLOCKS + b) * kMomentBlock;
      if (i0 >= n) break;
      const long long i = i0 + lane * PER;
      const int left = static_cast<int>(min(static_cast<long long>(PER), n - i));      // of this lane; may be negative
      const bool vec = left == PER && (low & 15u) == 0;
      const long long block = (t.at + i0) / kMomentBlock, s = t.at + i;
      float w[PER], g[PER], m[PER], v[PER];
      // gradient and weight; what is behind the end is 0
      if (vec) {
        const float4 w0 = *reinterpret_cast<const float4*>(t.weight + i), w1 = *reinterpret_cast<const float4*>(t.weight + i + 4);
        w[0] = w0.x; w[1] = w0.y; w[2] = w0.z; w[3] = w0.w; w[4] = w1.x; w[5] = w1.y; w[6] = w1.z; w[7] = w1.w;
        if (t.grad_bf16) {
          const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(t.grad) + i);
          const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            g[2 * j] = __uint_as_float(q[j] << 16);
            g[2 * j + 1] = __uint_as_float(q[j] & 0xFFFF0000u);
          }
        } else {
          const float* gp = static_cast<const float*>(t.grad) + i;
          const float4 g0 = *reinterpret_cast<const float4*>(gp), g1 = *reinterpret_cast<const float4*>(gp + 4);
          g[0] = g0.x; g[1] = g0.y; g[2] = g0.z; g[3] = g0.w; g[4] = g1.x; g[5] = g1.y; g[6] = g1.z; g[7] = g1.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          w[j] = j < left ? t.weight[i + j] : 0.f;
          g[j] = j >= left ? 0.f
                 : t.grad_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(t.grad)[i + j])
                               : static_cast<const float*>(t.grad)[i + j];
        }
      }
      // the moments' buffers are aligned and hold whole blocks, zeros behind the end
      if (BITS == 8) {
        const uint2 mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + s);
        const uint2 vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + s);
        const float ms = a.m_scale[block], vs = a.v_scale[block];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          m[j] = decode_m(((j < 4 ? mc.x : mc.y) >> (8 * (j & 3))) & 255u, ms);
          v[j] = decode_v(((j < 4 ? vc.x : vc.y) >> (8 * (j & 3))) & 255u, vs);
        }
      } else {
        const float4* mp = reinterpret_cast<const float4*>(static_cast<const float*>(a.m) + s);
        const float4* vp = reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + s);
        const float4 m0 = mp[0], m1 = mp[1], v0 = vp[0], v1 = vp[1];
        m[0] = m0.x; m[1] = m0.y; m[2] = m0.z; m[3] = m0.w; m[4] = m1.x; m[5] = m1.y; m[6] = m1.z; m[7] = m1.w;
        v[0] = v0.x; v[1] = v0.y; v[2] = v0.z; v[3] = v0.w; v[4] = v1.x; v[5] = v1.y; v[6] = v1.z; v[7] = v1.w;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float gj = __fmul_rn(g[j], a.grad_scale);
        m[j] = __fadd_rn(__fmul_rn(m[j], a.b1), __fmul_rn(gj, a.c1));
        v[j] = __fadd_rn(__fmul_rn(v[j], a.b2), __fmul_rn(__fmul_rn(gj, a.c2), gj));
        if (j >= left) m[j] = v[j] = 0.f;
        w[j] = w[j] * a.keep - rate * (m[j] / fmaf(sqrtf(v[j]), root, a.eps));
      }
      if (vec) {
        *reinterpret_cast<float4*>(t.weight + i) = make_float4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<float4*>(t.weight + i + 4) = make_float4(w[4], w[5], w[6], w[7]);
        if (t.param != nullptr)
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(t.param) + i) =
              make_uint4(pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3]), pack_bf16x2(w[4], w[5]), pack_bf16x2(w[6], w[7]));
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (j < left) {
            t.weight[i + j] = w[j];
            if (t.param != nullptr) static_cast<__nv_bfloat16*>(t.param)[i + j] = __float2bfloat16(w[j]);
          }
        }
      }
      if (BITS == 8) {
        const float ms = block_scale(m), vs = block_scale(v);
        const float dm = ms > 0.f ? ms : 1.f, dv = vs > 0.f ? vs : 1.f;
        uint32_t mc[2] = {0, 0}, vc[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t r = mix32(static_cast<uint32_t>(i + j) + t.seed);
          const uint32_t cm = encode_m(__fdiv_rn(fabsf(m[j]), dm), r & 0xFFFFu) | (m[j] < 0.f ? 128u : 0u);
          const uint32_t cv = encode_v(__fdiv_rn(v[j], dv), r >> 16);
          mc[j / 4] |= (cm & 255u) << (8 * (j & 3));
          vc[j / 4] |= (cv & 255u) << (8 * (j & 3));
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + s) = make_uint2(mc[0], mc[1]);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + s) = make_uint2(vc[0], vc[1]);
        if (lane == 0) {
          a.m_scale[block] = ms;
          a.v_scale[block] = vs;
        }
      } else {
        float4* mp = reinterpret_cast<float4*>(static_cast<float*>(a.m) + s);
        float4* vp = reinterpret_cast<float4*>(static_cast<float*>(a.v) + s);
        mp[0] = make_float4(m[0], m[1], m[2], m[3]);
        mp[1] = make_float4(m[4], m[5], m[6], m[7]);
        vp[0] = make_float4(v[0], v[1], v[2], v[3]);
        vp[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  }
}

template <bool SIGNED>
__global__ void __launch_bounds__(256)
moments_decode_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, float* __restrict__ out, long long n) {
  grid_begin(codes, scales);
  for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += 2048ll * gridDim.x) {
    const uint2 c = *reinterpret_cast<const uint2*>(codes + i);
    const float s = scales[i / kMomentBlock];
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t k = ((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 255u;
      x[j] = SIGNED ? decode_m(k, s) : decode_v(k, s);
    }
    __stcs(reinterpret_cast<float4*>(out + i), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4*>(out + i + 4), make_float4(x[4], x[5], x[6], x[7]));
  }
}

}  // namespace

int adamw_launch(AdamwTable& table, const AdamwArgs& a, int num_sms, cudaStream_t st) {
  long long chunks = 0;
  for (int i = 0; i < table.count; ++i) {
    table.first[i] = static_cast<int>(chunks);
    chunks += (table.t[i].n + CHUNK - 1) / CHUNK;
    if (chunks > INT32_MAX / 2) return -1;
  }
  table.first[table.count] = static_cast<int>(chunks);
  if (chunks == 0) return 0;
  const long long most = 8ll * num_sms;
  const dim3 grid(static_cast<unsigned>(chunks < most ? chunks : most));
  const cudaError_t e = a.m_scale != nullptr ? launch_overlapped(adamw_kernel<8>, grid, THREADS, 0, st, table, a)
                                             : launch_overlapped(adamw_kernel<32>, grid, THREADS, 0, st, table, a);
  return e == cudaSuccess ? 0 : -3;
}

int moments_decode(const void* codes, const float* scales, float* out, long long n, int is_signed, int num_sms, cudaStream_t st) {
  if (n == 0) return 0;
  const long long want = (n + 2047) / 2048, most = 16ll * num_sms;
  const dim3 grid(static_cast<unsigned>(want < most ? want : most));
  const auto kernel = is_signed ? moments_decode_kernel<true> : moments_decode_kernel<false>;
  return launch_overlapped(kernel, grid, 256, 0, st, static_cast<const uint8_t*>(codes), scales, out, n) == cudaSuccess ? 0 : -3;
}

}  // namespace piper
