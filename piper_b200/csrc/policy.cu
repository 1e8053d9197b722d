// Clipped policy loss with a KL term over a batch of tokens (packed.h).
//
// A token that counts has, with r = exp(logprob - old) and u = ref - logprob,
//   l = max(-A r, -A clip(r, low, high)) + beta (e^u - 1 - u),    dl/dlogprob = -A r [unless clipped] - beta (e^u - 1)
// and the loss is sum w l, w = 1 / (tokens that count), or 1 / (sequences that have such tokens x such tokens of its sequence).
// Differences are taken in 64 bits, where that of two fp32 numbers is exact but for far exponents, and compared with the logarithms of
// the borders there, so that a token is clipped or not as by the definition; r and e^u - 1 - u are fp32 numbers of those
// differences (the latter by its series near 0, where its terms cancel); sums are in 64 bits and in a fixed order.
//
// Some 20 bytes a token: bound by launches and latency.  One warp sums 128 tokens (of a block of the table, or just the next ones), one
// CTA adds the blocks' sums, those of sequences first where there is a table.  us a pass in a graph of 20 (launches overlap, caches are
// warm), forward, without and with sequences of some 1,000 tokens: 1,024 tokens 3.8 and 4.7 (one launch), 65,536 4.8 and 6.7, 131,072 5.3
// and 9.0, of which the bytes are 0.4; the gradient 2 to 4.  By itself and with cold caches (ncu) a launch takes 4 to 9.
#include "packed.h"

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int THREADS = 1024;

struct Sums {                  // of the tokens that count
  double loss, kl;
  int clipped, count;
  double unused;
};
static_assert(sizeof(Sums) == 32, "scratch is 32 bytes a block");

struct Token {
  float loss, kl, grad;
  bool clipped;
};

// e^u - 1 - u.  The series' next term is below 2^-26 of the sum where |u| < 0.5.  At u = inf the difference would be NaN.
__device__ __forceinline__ float exp_behind_linear(float u, float em1) {
  if (fabsf(u) >= 0.5f) return em1 == INFINITY ? em1 : em1 - u;
  float s = 1.f / 362880.f;
  s = fmaf(s, u, 1.f / 40320.f);
  s = fmaf(s, u, 1.f / 5040.f);
  s = fmaf(s, u, 1.f / 720.f);
  s = fmaf(s, u, 1.f / 120.f);
  s = fmaf(s, u, 1.f / 24.f);
  s = fmaf(s, u, 1.f / 6.f);
  s = fmaf(s, u, 0.5f);
  return s * u * u;
}

__device__ __forceinline__ Token token(const PolicyArgs& a, float logprob, float old, float adv, float ref) {
  Token t = {0.f, 0.f, 0.f, false};
  if (adv != 0.f) {                            // or a NaN
    const double d = static_cast<double>(logprob) - static_cast<double>(old);
    t.clipped = adv > 0.f ? d > a.log_high : adv < 0.f && d < a.log_low;      // a NaN has no border
    const float r = expf(static_cast<float>(d));
    t.loss = -adv * (t.clipped ? (adv > 0.f ? a.high : a.low) : r);
    t.grad = t.clipped ? 0.f : t.loss;
  }
  if (a.ref != nullptr) {
    const float u = static_cast<float>(static_cast<double>(ref) - static_cast<double>(logprob));
    const float em1 = expm1f(u);
    t.kl = exp_behind_linear(u, em1);
    if (a.kl_coef != 0.f) {
      t.loss = fmaf(a.kl_coef, t.kl, t.loss);
      t.grad = fmaf(-a.kl_coef, em1, t.grad);
    }
  }
  return t;
}

// First token and number of tokens (at most 128) of block i.
__device__ __forceinline__ void block_of(const PolicyArgs& a, const int4* table, long long i, long long* first, int* n, int* place) {
  if (table != nullptr) {
    const int4 e = __ldg(table + 1 + i);
    *first = e.x + e.z * 128;
    *n = min(128, e.y - e.z * 128);
    *place = e.w / 128 + e.z;
  } else {
    *first = i * 128;
    *n = static_cast<int>(min(128ll, a.T - i * 128));
    *place = static_cast<int>(i);
  }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// Tokens of a lane: every 32nd of a block, loaded together.
struct Loaded {
  float logprob[4], old[4], adv[4], ref[4];
  bool on[4];
};
__device__ __forceinline__ Loaded load(const PolicyArgs& a, long long first, int n, int lane) {
  Loaded x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long t = first + lane + 32 * j;
    const bool in = lane + 32 * j < n;
    x.on[j] = in && (a.mask == nullptr || a.mask[t] != 0);
    x.logprob[j] = in ? a.logprob[t] : 0.f;
    x.old[j] = in ? a.old[t] : 0.f;
    x.adv[j] = in ? a.adv[t] : 0.f;
    x.ref[j] = in && a.ref != nullptr ? a.ref[t] : 0.f;
  }
  return x;
}

__device__ long long blocks_in_use(const PolicyArgs& a, const int4* table) {
  if (table == nullptr) return a.blocks;
  const int4 header = __ldg(table);
  return header.z == a.T ? header.x : 0;       // of another batch: nothing counts
}

__device__ void sum_blocks(const PolicyArgs& a, const int4* table, Sums* sums) {
  const int lane = threadIdx.x & 31;
  const long long used = blocks_in_use(a, table), warps = static_cast<long long>(gridDim.x) * (blockDim.x / 32);
  for (long long i = static_cast<long long>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32; i < used; i += warps) {
    long long first;
    int n, place;
    block_of(a, table, i, &first, &n, &place);
    const Loaded x = load(a, first, n, lane);
    Sums s = {0., 0., 0, 0, 0.};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!x.on[j]) continue;
      const Token t = token(a, x.logprob[j], x.old[j], x.adv[j], x.ref[j]);
      s.loss += t.loss;
      s.kl += t.kl;
      s.clipped += t.clipped;
      ++s.count;
    }
    s.loss = warp_sum(s.loss);
    s.kl = warp_sum(s.kl);
    s.clipped = warp_sum(s.clipped);
    s.count = warp_sum(s.count);
    if (lane == 0) sums[place] = s;
  }
}

// One CTA: sums of the blocks, of sequences first where there is a table.
__device__ void add_blocks(const PolicyArgs& a, const int4* table, const Sums* sums, const PolicyOut& out) {
  __shared__ Sums parts[32];
  __shared__ int of_sequences[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
  const long long used = blocks_in_use(a, table);
  Sums s = {0., 0., 0, 0, 0.};
  int sequences = 0;
  if (table == nullptr) {
    for (long long i = threadIdx.x; i < used; i += blockDim.x) {
      const Sums b = sums[i];
      s.loss += b.loss;
      s.kl += b.kl;
      s.clipped += b.clipped;
      s.count += b.count;
    }
  } else {
    // The last entries, of place 0, are the sequences, those of most blocks first.  Long ones take a warp each, the others eight lanes.
    const int some = used > 0 ? __ldg(table).w : 0;
    const int4* const first = table + 1 + used - some;
    auto add = [&](const int4& e, int lanes, unsigned mask) {
      const int own = lane & (lanes - 1), place = e.w / 128, blocks = (e.y + 127) / 128;
      Sums q = {0., 0., 0, 0, 0.};
      for (int b = own; b < blocks; b += lanes) {
        const Sums v = sums[place + b];
        q.loss += v.loss;
        q.kl += v.kl;
        q.clipped += v.clipped;
        q.count += v.count;
      }
      for (int o = lanes / 2; o > 0; o >>= 1) {
        q.loss += __shfl_xor_sync(mask, q.loss, o);
        q.kl += __shfl_xor_sync(mask, q.kl, o);
        q.clipped += __shfl_xor_sync(mask, q.clipped, o);
        q.count += __shfl_xor_sync(mask, q.count, o);
      }
      if (own != 0) return;
      out.weight[1 + place] = q.count > 0 ? 1.f / static_cast<float>(q.count) : 0.f;
      if (q.count == 0) return;
      s.loss += q.loss / q.count;
      s.kl += q.kl / q.count;
      s.clipped += q.clipped;
      s.count += q.count;
      ++sequences;
    };
    constexpr int kLong = 64 * 128;
    for (int i = warp; i < some; i += warps) {
      const int4 e = __ldg(first + i);
      if (e.y <= kLong) break;
      add(e, 32, 0xffffffffu);
    }
    __syncwarp();
    for (int i = threadIdx.x / 8; i < some; i += blockDim.x / 8) {
      const int4 e = __ldg(first + i);
      if (e.y <= kLong) add(e, 8, 0xffu << (lane & 24));
    }
    __syncwarp();
  }
  s.loss = warp_sum(s.loss);
  s.kl = warp_sum(s.kl);
  s.clipped = warp_sum(s.clipped);
  s.count = warp_sum(s.count);
  sequences = warp_sum(sequences);
  if (lane == 0) {
    parts[warp] = s;
    of_sequences[warp] = sequences;
  }
  __syncthreads();
  if (warp != 0) return;
  s = lane < warps ? parts[lane] : Sums{0., 0., 0, 0, 0.};
  sequences = warp_sum(lane < warps ? of_sequences[lane] : 0);
  s.loss = warp_sum(s.loss);
  s.kl = warp_sum(s.kl);
  s.clipped = warp_sum(s.clipped);
  s.count = warp_sum(s.count);
  if (lane != 0) return;
  const int n = max(1, table == nullptr ? s.count : sequences);
  *out.loss = static_cast<float>(s.loss / n);
  *out.kl = static_cast<float>(s.kl / n);
  *out.clipped = static_cast<float>(static_cast<double>(s.clipped) / max(1, s.count));
  out.weight[0] = static_cast<float>(1. / n);
}

// The table is read by __ldg, often right behind the launch that writes it: by the pointer that comes out of the wait alone.
__device__ __forceinline__ const int4* begin_with_table(const PolicyArgs& a) {
  const int4* table = reinterpret_cast<const int4*>(a.table);
  grid_begin(table);
  return a.table == nullptr ? nullptr : table;
}

__global__ void __launch_bounds__(THREADS) policy_one_kernel(const PolicyArgs a, const PolicyOut out, Sums* sums) {
  const int4* const table = begin_with_table(a);
  sum_blocks(a, table, sums);
  __syncthreads();
  add_blocks(a, table, sums, out);
}

__global__ void __launch_bounds__(256) policy_sums_kernel(const PolicyArgs a, Sums* sums) {
  const int4* const table = begin_with_table(a);
  sum_blocks(a, table, sums);
}

__global__ void __launch_bounds__(THREADS) policy_add_kernel(const PolicyArgs a, const PolicyOut out, Sums* sums) {
  const int4* const table = begin_with_table(a);
  add_blocks(a, table, sums, out);
}

__global__ void __launch_bounds__(256) policy_bwd_kernel(const PolicyArgs a, const float* weight, const float* d_loss,
                                                         float* d) {
  const int4* const table = begin_with_table(a);
  const int lane = threadIdx.x & 31;
  const long long used = blocks_in_use(a, table), warps = static_cast<long long>(gridDim.x) * (blockDim.x / 32);
  const float up = *d_loss * weight[0];
  for (long long i = static_cast<long long>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32; i < used; i += warps) {
    long long first;
    int n, place;
    block_of(a, table, i, &first, &n, &place);
    const Loaded x = load(a, first, n, lane);
    const float w = table == nullptr ? up : up * weight[1 + __ldg(table + 1 + i).w / 128];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (lane + 32 * j >= n) continue;
      d[first + lane + 32 * j] = x.on[j] ? token(a, x.logprob[j], x.old[j], x.adv[j], x.ref[j]).grad * w : 0.f;
    }
  }
  if (table == nullptr) return;
  const int4 header = __ldg(table);            // tokens behind the last sequence
  for (long long t = (header.z == a.T ? header.y : 0) + static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; t < a.T;
       t += static_cast<long long>(gridDim.x) * blockDim.x)
    d[t] = 0.f;
}

// One CTA does all up to here, a block a warp.  us a pass in a graph of 20 in one launch and in two, of which the second costs the host
// 2.5: 128 tokens 3.5 and 4.1, 1,024 3.8 and 4.4, 4,096 5.2 and 4.4.  (One cluster of eight CTAs: 16,384 tokens 6.1 and 4.5, 65,536 8.9
// and 4.8.)
constexpr long long kOneCtaBlocks = THREADS / 32;

}  // namespace

int policy_fwd(const PolicyArgs& a, const PolicyOut& out, void* scratch, int num_sms, cudaStream_t st) {
  if (a.T < 0 || a.blocks < 0 || a.blocks > INT32_MAX / 128 || (a.table != nullptr && a.T > kMaxPackedTokens)) return -1;
  Sums* const sums = static_cast<Sums*>(scratch);
  if (a.blocks <= kOneCtaBlocks) {
    launch_overlapped(policy_one_kernel, 1, THREADS, 0, st, a, out, sums);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
  }
  const long long ctas = (a.blocks + 7) / 8;
  launch_overlapped(policy_sums_kernel, static_cast<unsigned>(ctas < 8ll * num_sms ? ctas : 8ll * num_sms), 256, 0, st, a, sums);
  if (cudaGetLastError() != cudaSuccess) return -3;
  launch_overlapped(policy_add_kernel, 1, THREADS, 0, st, a, out, sums);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int policy_bwd(const PolicyArgs& a, const float* weight, const float* d_loss, float* d, int num_sms, cudaStream_t st) {
  if (a.T < 0 || a.blocks < 0 || a.blocks > INT32_MAX / 128 || (a.table != nullptr && a.T > kMaxPackedTokens)) return -1;
  if (a.T == 0) return 0;
  // A warp for every block, of which short sequences have more than their tokens say (600 tokens in 500 sequences: CTAs by tokens
  // 44 us, by blocks 2.3), and for every 128 tokens behind the last sequence.
  const long long of_tokens = (a.T + 127) / 128, ctas = ((a.blocks > of_tokens ? a.blocks : of_tokens) + 7) / 8;
  launch_overlapped(policy_bwd_kernel, static_cast<unsigned>(ctas < 8ll * num_sms ? ctas : 8ll * num_sms), 256, 0, st, a, weight, d_loss,
                    d);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace piper
