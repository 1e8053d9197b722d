// Balance loss of a router (packed.h): with p = softmax(logits) of the N tokens that count, P_e their mean probability of expert e and
// f_e = counts_e / (N k) the share of the choices that went to it,
//   loss = E sum_e f_e P_e,    dloss/dlogit_te = p_te (c_e - sum_j p_tj c_j),    c_e = E f_e / N.
// The counts have no gradient.  A row without a finite logit has probabilities 0 and no gradient.
//
// Forward: one read of the logits and choices.  Lanes hold eight neighbouring experts of a row (one 16-byte vector of bf16, two of fp32),
// so a warp works on 256 / E rows at once, and each lane adds up the probabilities of its experts over its rows in fp32; choices are
// counted in shared memory.  A CTA leaves its sums, one CTA adds those of all in a fixed order in 64 bits: behind a
// cluster barrier where one cluster is enough for the rows, in a second launch otherwise.  Backward: the probabilities again, one
// read and one write of the logits.  us of the three kernels by themselves with cold caches (ncu): 16,384 x 128 bf16 8.4, 15.7 and 8.2
// (0.7, 0 and 1.3 at the measured bandwidth), 131,072 x 64 18, 10 and 16 (3.3, 0 and 5.1); in a graph of 20 passes (launches overlap,
// caches are warm) 15 forward and 6 backward, 19 and 13: launches and latencies, that of the one CTA that adds above all.
#include "packed.h"

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int CLUSTER = 8;

template <bool F32>
__device__ __forceinline__ void load8(const void* logits, long long at, int left, bool vector, float (&x)[8]) {
  if (vector && left >= 8) {
    if constexpr (F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(logits) + at);
      const float4 a = p[0], b = p[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(logits) + at);
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(h[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = -INFINITY;
    if (i < left) {
      if constexpr (F32) x[i] = static_cast<const float*>(logits)[at + i];
      else x[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[at + i]);
    }
  }
}

// Probabilities of a row in place of its logits; the row is with `lanes` neighbouring lanes.
__device__ __forceinline__ void softmax8(float (&x)[8], int lanes) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
  for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;             // nothing is left: all become 0
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = expf(x[i] - top);
    sum += x[i];
  }
  for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= inv;
}

// scratch: per CTA E + 1 floats (sums of probabilities) and E + 1 ints (counts; tokens that count)
__device__ __forceinline__ float* sums_of(void* scratch, int E, int cta) {
  return static_cast<float*>(scratch) + static_cast<long long>(cta) * 2 * (E + 1);
}

template <bool F32>
__device__ void sum_rows(const BalanceArgs& a, int lanes, void* scratch) {
  __shared__ float probs[WARPS][kMaxBalanceExperts];
  __shared__ int counts[kMaxBalanceExperts + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= a.E; e += THREADS) counts[e] = 0;
  __syncthreads();
  const int per_warp = 32 / lanes, e0 = (lane & (lanes - 1)) * 8, left = a.E - e0;
  const bool vector = a.E % 8 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  const long long step = static_cast<long long>(gridDim.x) * WARPS * per_warp;
  float sum[8] = {};
  int tokens = 0;
  for (long long t0 = (static_cast<long long>(blockIdx.x) * WARPS + warp) * per_warp; t0 < a.T; t0 += 2 * step) {
    const long long t[2] = {t0 + lane / lanes, t0 + step + lane / lanes};     // two rows at a time: their loads overlap
    bool on[2];
    float x[2][8] = {};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      on[r] = t[r] < a.T && (a.mask == nullptr || a.mask[t[r]] != 0);
      if (on[r]) load8<F32>(a.logits, t[r] * a.E + e0, left, vector, x[r]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      softmax8(x[r], lanes);
      if (!on[r]) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += x[r][i];
      tokens += e0 == 0;
    }
  }
  // choices: all threads over the rows' k, which lie one behind the other
  const unsigned n = static_cast<unsigned>(a.T * a.k), stride = gridDim.x * THREADS;      // below 2^31
  for (unsigned i = blockIdx.x * THREADS + threadIdx.x; i < n; i += stride) {
    if (a.mask != nullptr && a.mask[i / a.k] == 0) continue;
    const int e = a.idx[i];
    if (e >= 0 && e < a.E) atomicAdd(&counts[e], 1);
    else report_bad_argument(a.status, 61, e, a.E);
  }
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  if (lane == 0) atomicAdd(&counts[a.E], tokens);
  // over the rows of a warp, then over the warps
#pragma unroll
  for (int i = 0; i < 8; ++i)
    for (int o = lanes; o < 32; o <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  if (lane < lanes) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) probs[warp][e0 + i] = sum[i];
  }
  __syncthreads();
  float* const mine = sums_of(scratch, a.E, blockIdx.x);
  for (int e = threadIdx.x; e <= a.E; e += THREADS) {
    float s = 0.f;
    if (e < a.E)
      for (int w = 0; w < WARPS; ++w) s += probs[w][e];
    mine[e] = s;
    reinterpret_cast<int*>(mine)[a.E + 1 + e] = counts[e];
  }
}

constexpr int ADD_THREADS = 1024;

__device__ void add_rows(const BalanceArgs& a, int ctas, void* scratch, float* loss, int* counts, float* prob, float* factor) {
  __shared__ double sums[ADD_THREADS];
  __shared__ int chosen[ADD_THREADS];
  __shared__ double terms[kMaxBalanceExperts];
  __shared__ int tokens;
  // Neighbouring threads have neighbouring experts (the last place: tokens that count) of one of `parts` shares of the CTAs.
  const int width = a.E + 1, parts = blockDim.x / width;
  const int part = threadIdx.x / width, e = threadIdx.x - part * width;
  double p = 0.;
  int count = 0;
  if (part < parts) {
    const float* s = sums_of(scratch, a.E, part) + e;
    const long long step = 2ll * width * parts;
#pragma unroll 8
    for (int c = part; c < ctas; c += parts, s += step) {
      p += s[0];
      count += reinterpret_cast<const int*>(s)[width];
    }
    sums[threadIdx.x] = p;
    chosen[threadIdx.x] = count;
  }
  __syncthreads();
  if (threadIdx.x < width) {
    for (int i = 1; i < parts; ++i) {
      p += sums[i * width + e];
      count += chosen[i * width + e];
    }
    if (e == a.E) tokens = count;
  }
  __syncthreads();
  const double n = max(1, tokens);
  if (threadIdx.x < a.E) {
    const double f = count * (a.E / (n * a.k));
    counts[e] = count;
    prob[e] = static_cast<float>(p / n);
    factor[e] = static_cast<float>(f / n);
    terms[e] = f * (p / n);
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  double sum = 0.;
  for (int i = threadIdx.x; i < a.E; i += 32) sum += terms[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x == 0) *loss = static_cast<float>(sum);
}

template <bool F32>
__global__ void __launch_bounds__(THREADS)
balance_cluster_kernel(const BalanceArgs a, int lanes, void* scratch, float* loss, int* counts, float* prob, float* factor) {
  grid_begin();
  sum_rows<F32>(a, lanes, scratch);
  __threadfence();
  cluster_sync();
  if (blockIdx.x == 0) add_rows(a, gridDim.x, scratch, loss, counts, prob, factor);
}

template <bool F32>
__global__ void __launch_bounds__(THREADS) balance_sums_kernel(const BalanceArgs a, int lanes, void* scratch) {
  grid_begin();
  sum_rows<F32>(a, lanes, scratch);
}

__global__ void __launch_bounds__(ADD_THREADS)
balance_add_kernel(const BalanceArgs a, int ctas, void* scratch, float* loss, int* counts, float* prob, float* factor) {
  grid_begin();
  add_rows(a, ctas, scratch, loss, counts, prob, factor);
}

template <bool F32>
__global__ void __launch_bounds__(THREADS)
balance_bwd_kernel(const BalanceArgs a, int lanes, const float* factor, const float* d_loss, void* d) {
  grid_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per_warp = 32 / lanes, e0 = (lane & (lanes - 1)) * 8, left = a.E - e0;
  const bool vector = a.E % 8 == 0 && (reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(d)) % 16 == 0;
  const float up = *d_loss;
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = i < left ? factor[e0 + i] * up : 0.f;
  const long long step = static_cast<long long>(gridDim.x) * WARPS * per_warp;
  for (long long t0 = (static_cast<long long>(blockIdx.x) * WARPS + warp) * per_warp; t0 < a.T; t0 += step) {
    const long long t = t0 + lane / lanes, at = t * a.E + e0;
    const bool on = t < a.T && (a.mask == nullptr || a.mask[t] != 0);
    float x[8] = {};
    if (on) load8<F32>(a.logits, at, left, vector, x);
    softmax8(x, lanes);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(x[i], c[i], dot);
    for (int o = lanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = on ? x[i] * (c[i] - dot) : 0.f;
    if (t >= a.T || left <= 0) continue;
    if (vector) {
      if constexpr (F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(d) + at);
        p[0] = make_float4(x[0], x[1], x[2], x[3]);
        p[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(d) + at) =
            make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= left) continue;
        if constexpr (F32) static_cast<float*>(d)[at + i] = x[i];
        else static_cast<__nv_bfloat16*>(d)[at + i] = __float2bfloat16(x[i]);
      }
    }
  }
}

// Lanes of a row: a power of two.
int lanes_of(int E) {
  int lanes = 1;
  while (lanes * 8 < E) lanes *= 2;
  return lanes;
}

bool takes(const BalanceArgs& a) {
  return a.E >= 1 && a.E <= kMaxBalanceExperts && a.k >= 1 && a.k <= a.E && a.T >= 0 && a.T * a.k <= INT32_MAX;
}

// Up to this many logits one cluster is enough.  us a pass in a graph of 20 as one cluster and in two launches, of which the second costs
// the host 2.5: 512 x 8 7.1 and 7.4, 1,024 x 64 6.8 and 6.6, 2,048 x 64 8.6 and 7.0, 1,024 x 128 9.2 and 7.8.
constexpr long long kClusterLogits = 1 << 16;

long long row_ctas(long long T, int E) {
  const long long rows = WARPS * (32 / lanes_of(E));
  return (T + rows - 1) / rows;
}

}  // namespace

int balance_ctas(long long T, int E, int num_sms) {
  const long long ctas = row_ctas(T, E);
  if (ctas <= 1) return 1;
  if (T * E <= kClusterLogits) return CLUSTER;
  return static_cast<int>(ctas < 2ll * num_sms ? ctas : 2ll * num_sms);
}

int balance_fwd(const BalanceArgs& a, float* loss, int* counts, float* prob, float* factor, void* scratch, int num_sms, cudaStream_t st) {
  if (!takes(a)) return -1;
  const int lanes = lanes_of(a.E), ctas = balance_ctas(a.T, a.E, num_sms);
  if (ctas <= CLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = ctas;
    cfg.blockDim = THREADS;
    cfg.stream = st;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, a.f32 ? balance_cluster_kernel<true> : balance_cluster_kernel<false>, a, lanes, scratch, loss, counts,
                       prob, factor);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
  }
  launch_overlapped(a.f32 ? balance_sums_kernel<true> : balance_sums_kernel<false>, ctas, THREADS, 0, st, a, lanes, scratch);
  if (cudaGetLastError() != cudaSuccess) return -3;
  launch_overlapped(balance_add_kernel, 1, ADD_THREADS, 0, st, a, ctas, scratch, loss, counts, prob, factor);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int balance_bwd(const BalanceArgs& a, const float* factor, const float* d_loss, void* d, int num_sms, cudaStream_t st) {
  if (!takes(a)) return -1;
  if (a.T == 0) return 0;
  const long long ctas = row_ctas(a.T, a.E);
  launch_overlapped(a.f32 ? balance_bwd_kernel<true> : balance_bwd_kernel<false>,
                    static_cast<unsigned>(ctas < 8ll * num_sms ? ctas : 8ll * num_sms), THREADS, 0, st, a, lanes_of(a.E), factor, d_loss, d);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace piper
