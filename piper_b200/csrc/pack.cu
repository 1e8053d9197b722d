// The table of a packed batch (packed.h), by one CTA: a counting sort of the sequences, or of the groups of short ones, by their
// blocks of 128 rows.  Groups are formed greedily, from the first sequence of each of 32 parts on, by a warp each.
//
// With cnt[i] the number of sequences that have more than i blocks, the blocks with place i in their sequence come behind
// those of all later places, base[i] = sum_{j > i} cnt[j], and among them in the order of the sequences by falling number
// of blocks: the first cnt[i] of that order are those that have such a block.  Equal ones keep their order, so the table of a batch
// is always the same.  Bound by the latency of its few passes; done once for a batch, whatever the number of layers that use it.
#include "packed.h"

#include <atomic>

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int PACK_THREADS = 1024;

// Sums of the values of the threads before this one, and of all.
__device__ __forceinline__ int scan_before(int v, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                             // the sums of the call before have been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < PACK_THREADS / 32; ++w) {
    const int s = warp_sums[w];
    before += w < warp ? s : 0;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// a[i] becomes the sum of a[j] over j > i, or j >= i; returns the sum of all.
__device__ int sum_from_the_end(int* a, int m, bool with_own, int* warp_sums) {
  const int per = (m + PACK_THREADS - 1) / PACK_THREADS;
  const int hi = m - static_cast<int>(threadIdx.x) * per, lo = max(0, hi - per);
  int own = 0;
  for (int i = hi - 1; i >= lo; --i) own += a[i];
  int total;
  int sum = scan_before(own, warp_sums, &total);
  for (int i = hi - 1; i >= lo; --i) {
    const int v = a[i];
    a[i] = with_own ? sum + v : sum;
    sum += v;
  }
  __syncthreads();
  return total;
}

// Sequences [s0, s1) of a part, by one warp: items[s] becomes the rows of a sequence or, with kGrouped added, of the group that it
// begins; -(first sequence of its group) - 1 for the others of a group; 0 without rows.
constexpr int kGrouped = 1 << 30;
__device__ void group_sequences(const int* cu, int s0, int s1, int* items) {
  const int lane = threadIdx.x & 31;
  for (int s = s0; s < s1;) {
    const int a = cu[s], len = cu[s + 1] - a;
    if (len == 0 || len > 128) {
      if (lane == 0) items[s] = len;
      ++s;
      continue;
    }
    int end = s, some = 0;                     // behind the group, sequences of it that have rows
    while (end < s1) {
      const int t = end + 1 + lane;
      const bool fits = t <= s1 && cu[t] - a <= 128;
      const unsigned in = __ballot_sync(0xffffffffu, fits);
      some += __popc(__ballot_sync(0xffffffffu, fits && cu[t] > cu[t - 1]));
      if (fits && t - 1 > s) items[t - 1] = cu[t] > cu[t - 1] ? -s - 1 : 0;
      end += __popc(in);
      if (in != 0xffffffffu) break;
    }
    if (lane == 0) items[s] = cu[end] - a + (some > 1 ? kGrouped : 0);
    s = end;
  }
}

// own, items and pads (scratch) are null without groups.
__global__ void __launch_bounds__(PACK_THREADS)
pack_table_kernel(const int* __restrict__ cu, int n, int T, int blocks, int4* table, uchar2* own, int* items, int* pads, int* status) {
  grid_begin(cu);
  extern __shared__ int places[];              // base [m], next [m]
  __shared__ int warp_sums[PACK_THREADS / 32];
  static_assert(kGroupChunks <= PACK_THREADS / 32, "a warp for every part");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int m = (T + 127) / 128;               // blocks that a sequence may have
  int* const base = places;
  int* const next = places + m;
  for (int i = threadIdx.x; i < m; i += PACK_THREADS) base[i] = 0;
  int bad = 0;
  if (threadIdx.x == 0 && cu[0] != 0) {
    bad = 1;
    report_bad_argument(status, 51, 0, cu[0]);
  }
  for (int s = threadIdx.x; s < n; s += PACK_THREADS) {
    const int a = cu[s], b = cu[s + 1];
    if (a < 0 || b < a || b > T) {
      bad = 1;
      report_bad_argument(status, 51, s + 1, b);
    }
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) table[0] = make_int4(0, 0, T, 0);
    return;
  }
  if (items != nullptr) {
    const int chunk = group_chunk(n);
    if (warp < kGroupChunks && static_cast<long long>(warp) * chunk < n)
      group_sequences(cu, warp * chunk, static_cast<int>(min(static_cast<long long>(n), (warp + 1ll) * chunk)), items);
    __syncthreads();
  }
  auto rows_of = [&](int s) { return items == nullptr ? cu[s + 1] - cu[s] : max(items[s], 0) & ~kGrouped; };
  for (int s = threadIdx.x; s < n; s += PACK_THREADS) {
    const int len = rows_of(s);
    if (len > 0) atomicAdd(&base[(len + 127) / 128 - 1], 1);
  }
  __syncthreads();
  sum_from_the_end(base, m, true, warp_sums);  // base[i] = cnt[i]
  // of the sequences of v blocks the first comes behind all of more: next[v - 1] = cnt[v]
  for (int i = threadIdx.x; i < m; i += PACK_THREADS) next[i] = i + 1 < m ? base[i + 1] : 0;
  __syncthreads();
  const int some = m > 0 ? base[0] : 0;        // sequences that have rows; read before the next sums
  __syncthreads();
  const int used = sum_from_the_end(base, m, false, warp_sums);
  if (threadIdx.x == 0) table[0] = used <= blocks ? make_int4(used, cu[n], T, some) : make_int4(0, 0, T, 0);
  if (used > blocks) {                         // the caller's memory is for fewer: its number did not come from these sequences
    if (threadIdx.x == 0) report_bad_argument(status, 52, used, blocks);
    return;
  }
  int before = 0;                              // blocks of the sequences of earlier rounds
  for (int s0 = 0; s0 < n; s0 += PACK_THREADS) {
    const int s = s0 + threadIdx.x;
    const int start = s < n ? cu[s] : 0, len = s < n ? rows_of(s) : 0, nb = (len + 127) / 128;
    int all;
    int first = (before + scan_before(nb, warp_sums, &all)) * 128;
    before += all;
    if (items != nullptr && s < n) {
      pads[s] = first;
      if (items[s] > 0 && (items[s] & kGrouped) != 0) first += kGroup;
    }
    int rank = 0;
    for (int w = 0; w < PACK_THREADS / 32 && s0 + w * 32 < n; ++w) {
      if (warp == w) {
        const unsigned same = __match_any_sync(0xffffffffu, nb);
        const int leader = __ffs(same) - 1;
        int at = 0;
        if (lane == leader && nb > 0) {
          at = next[nb - 1];
          next[nb - 1] = at + __popc(same);
        }
        rank = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
      }
      __syncthreads();
    }
    for (int j = 0; j < 32; ++j) {             // a warp writes the blocks of its sequences one sequence after the other
      const int blocks_j = __shfl_sync(0xffffffffu, nb, j), start_j = __shfl_sync(0xffffffffu, start, j);
      const int len_j = __shfl_sync(0xffffffffu, len, j), first_j = __shfl_sync(0xffffffffu, first, j);
      const int rank_j = __shfl_sync(0xffffffffu, rank, j);
      for (int i = lane; i < blocks_j; i += 32)
        table[1 + base[i] + rank_j] = make_int4(start_j, len_j, i, first_j);
    }
  }
  if (items == nullptr) return;
  __syncthreads();
  // first and last rows of the sequences in groups; a warp takes a sequence
  for (int s = warp; s < n; s += PACK_THREADS / 32) {
    const int item = items[s];
    if (item == 0 || (item > 0 && (item & kGrouped) == 0)) continue;
    const int leader = item < 0 ? -item - 1 : s, off = cu[s] - cu[leader], len = cu[s + 1] - cu[s];
    for (int i = lane; i < len; i += 32)
      own[pads[leader] + off + i] = make_uchar2(static_cast<unsigned char>(off), static_cast<unsigned char>(off + len - 1));
  }
}

}  // namespace

int pack_table(const int* cu, int n, int T, int blocks, int* table, unsigned char* own, int* scratch, int* status, cudaStream_t st) {
  if (n < 0 || T < 0 || T > kMaxPackedTokens || blocks < 0) return -1;
  const int smem = (T + 127) / 128 * 2 * static_cast<int>(sizeof(int));
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return -2;
  static std::atomic<bool> configured[64];
  if (!configured[device].load()) {
    if (cudaFuncSetAttribute(pack_table_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPackedTokens / 128 * 8) !=
        cudaSuccess)
      return -2;
    configured[device].store(true);
  }
  launch_overlapped(pack_table_kernel, 1, PACK_THREADS, smem, st, cu, n, T, blocks, reinterpret_cast<int4*>(table),
                    reinterpret_cast<uchar2*>(own), own != nullptr ? scratch : nullptr, own != nullptr ? scratch + n : nullptr, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace piper
