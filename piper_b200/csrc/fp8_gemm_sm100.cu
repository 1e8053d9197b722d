// Products of e4m3 operands with a power-of-two scale for every row and 128 columns: C[M, N] = A[M, K] B[N, K]^T, bf16 or added
// into fp32.
//
//   C[m, n] = sum over blocks k of 2^(ea[m, k] + eb[n, k]) sum over the block of a[m, i] b[n, i]
//
// The tensor core multiplies with the scales itself (tcgen05.mma kind::mxf8f6f4 with block_scale, which takes a scale for
// every 32 of the contraction: four instructions in a row take the same one) and keeps the sum in fp32 in tensor memory, so
// no partial sum leaves it before the end.  Scaling by powers of two is exact; the sum is a little coarser than single additions in fp32:
// within 2^-22 of the sum of the magnitudes for every 32 of the contraction, which is added at once.  A contraction of 28672
// differs from an fp32 sum by 1.1e-4 of the result's norm, a last bit of bf16 in one of a thousand elements; both are 1.66e-3 of the norm,
// bf16's own rounding, from the exact product.
//
// Persistent CTAs, each by itself or in pairs on two neighbouring SMs (cta_group::2), walk tiles of 128 rows a CTA and 32 to 224 columns.
// Roles by warp:
//   warp 0       TMA producer: a ring of shared-memory stages of 128 x 128-byte operand boxes in 128-byte swizzle; hands out tiles.
//   warp 1       MMA issuer (first CTA of a pair, for both), into one of two accumulators.
//   warp 2       tensor memory allocation.
//   warps 4-11   epilogue: accumulator to bf16 or fp32, through shared memory, TMA store or reduce-add.
//   warps 12-15  scales: words of four blocks from global memory into tensor memory, one warp for each quarter of its lanes, which
//                all hold the same: row r of A in lane r % 32 of column r / 32, rows of B likewise behind them.
// Tensor memory: two accumulators of 224 columns, then four slots of 16 columns for the scales of four blocks (4 for 128 rows of A,
// up to 7 for B).  256 columns would leave no room for the scales beside a second accumulator.
//
// A stage holds one block of the contraction, or two.
//
// What bounds it: a block of 128 of a 256 x 224 tile of a pair takes 448 cycles of MMA and loads 30 KiB into each SM, 472 cycles at
// the 65 bytes per cycle that an SM takes from L2.  4096 x 28672 x 4096: 306-309 us by itself (3.1 PFLOP/s, tensor pipe 88 % busy),
// 316-327 in a loop of some; in a long loop the clock falls under the power limit, to some 390 us.  Few rows: a block's issue, see
// two_blocks().
//
// All waits are bounded; on expiry the kernel records a status code, drains its copies, frees its tensor memory and returns.
#include "fp8.h"

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdlib>
#include <mutex>
#include <unordered_map>

#include "gemm_sm100.h"
#include "ptx.cuh"

namespace piper {
namespace {

constexpr int BM = 128;
constexpr int BK = kFp8Group;                  // elements and bytes
constexpr int UMMA_K = 32;
constexpr int A_STAGE_BYTES = BM * BK;
constexpr int MAX_WIDTH = 224;
constexpr int MAX_STAGES = 8;
constexpr int OPERAND_BYTES = 196608;
constexpr int EPI_WARPS = 8;
constexpr int SCALE_WARPS = 4;
constexpr int NUM_THREADS = 128 + 32 * (EPI_WARPS + SCALE_WARPS);
constexpr int C_STAGE_BYTES = 4096;
constexpr int BAR_OFF = OPERAND_BYTES + EPI_WARPS * C_STAGE_BYTES;
constexpr int SMEM_BYTES = BAR_OFF + 768 + 1024;
constexpr int RING = 16;
constexpr int SLOTS = 4;
constexpr uint32_t SLOT_COLUMN = 2 * MAX_WIDTH, SLOT_COLUMNS = 16;
static_assert(SLOT_COLUMN + SLOTS * SLOT_COLUMNS <= 512, "tensor memory");

struct Bars {
  uint64_t full[MAX_STAGES];
  uint64_t empty[MAX_STAGES];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint64_t scale_full[SLOTS];
  uint64_t scale_empty[SLOTS];
  uint64_t tile_full[RING];
  int tile[RING][4];
  uint32_t tmem_base;
};
static_assert(sizeof(Bars) <= 768 && offsetof(Bars, tile) % 16 == 0 && SMEM_BYTES <= 232448, "shared memory");

struct Params {
  const uint32_t* a_scales;
  const uint32_t* b_scales;
  int M, N, K;
  int a_pad, b_pad;   // rows of a group's words
  int width;
  int a_rows;         // rows of an A box: 128, or fewer where a CTA by itself has all rows
  int stages;
  int band;
  int* status;
  int slot;           // counter of the stream, or -1: tiles in a fixed order
};

// Counters of tiles, one per stream: a launch draws behind its wait for the kernel before it, whose last draw has rearmed the counter.
// They are the module's own, so every device has its zeros without an allocation.
constexpr unsigned SCHED_SLOTS = 1024;
__device__ int sched_slots[SCHED_SLOTS];

// D[tmem] (+)= (A * scales) * (B * scales), e4m3 inputs.
template <int CTAS>
__device__ __forceinline__ void umma_scaled(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a,
                                            uint32_t scale_b, uint32_t accumulate) {
  if (CTAS == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(scale_a), "r"(scale_b)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(scale_a), "r"(scale_b)
        : "memory");
}

// e4m3 x e4m3, both K-major, scales as exponents; bits 4-5 and 29-30 say which byte of the scales' words belongs to the block.
__device__ __forceinline__ uint32_t scaled_idesc(int m, int n, uint32_t byte) {
  return byte << 4 | static_cast<uint32_t>(n >> 3) << 17 | 1u << 23 | static_cast<uint32_t>(m >> 4) << 24 | byte << 29;
}

constexpr uint32_t NEXT_BYTE = 1u << 4 | 1u << 29;

__device__ __forceinline__ void tmem_st_32x4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int CTAS, bool F32, int BLOCKS>
__global__ void __launch_bounds__(NUM_THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_c, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  Bars* bars = reinterpret_cast<Bars*>(smem + BAR_OFF);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
  const int width = p.width;
  const int b_rows = width / CTAS;
  const int block_bytes = A_STAGE_BYTES + b_rows * BK, stage_bytes = block_bytes * BLOCKS;
  const int stages = p.stages;
  const int tiles_m = (p.M + BM * CTAS - 1) / (BM * CTAS);
  const int tiles_n = (p.N + width - 1) / width;
  const int num_tiles = tiles_m * tiles_n;
  const int k_blocks = (p.K + BK - 1) / BK;
  const bool n_fast = tiles_n < tiles_m;

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&bars->acc_full[a], 1);
      mbar_init(&bars->acc_empty[a], EPI_WARPS * CTAS);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&bars->scale_full[s], SCALE_WARPS * CTAS);
      mbar_init(&bars->scale_empty[s], 1);
    }
    for (int i = 0; i < RING; ++i) mbar_init(&bars->tile_full[i], 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_c);
  }
  if (warp == 2) {
    tmem_alloc_n<CTAS>(&bars->tmem_base, 512);
    tmem_relinquish_n<CTAS>();
  }
  // The first tile is the unit's own, later ones come from a counter, drawn while the last stage of the tile before is waited for.  With
  // the GPU to itself that changes little (4096 x 4096 x 28672 347 us, 353 in a fixed order; 2048 x 8192 x 992 17.7 and 17.2), but beside
  // another kernel that keeps 8 SMs: 4096 x 28672 x 4096 316 us and 525, 4096 x 4096 x 4096 66 and 81.
  const int units = static_cast<int>(gridDim.x) / CTAS;
  const bool draws = p.slot >= 0 && num_tiles > units;
  int* const counter = sched_slots + (draws ? p.slot : 0);
  grid_wait();
  tc_fence_before();
  if (CTAS == 2) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);

  // The dimension with fewer tiles is walked fastest, in bands where its operand does not stay in L2.
  auto coords = [&](int tile, int& tm, int& tn) {
    const int fast = n_fast ? tiles_n : tiles_m, slow = n_fast ? tiles_m : tiles_n;
    const int b = tile / (p.band * slow), f0 = b * p.band;
    const int bw = min(p.band, fast - f0), r = tile - f0 * slow;
    const int f = f0 + r % bw, sl = r / bw;
    tm = n_fast ? sl : f;
    tn = n_fast ? f : sl;
  };
  auto tile_at = [&](uint32_t n, int& tile) -> bool {
    if (!__all_sync(0xffffffffu, mbar_wait(&bars->tile_full[n % RING], (n / RING) & 1, p.status))) return false;
    tile = *reinterpret_cast<volatile int*>(&bars->tile[n % RING]);
    return true;
  };

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer (both CTAs of a pair load their own halves)
    const int loaded = p.a_rows * BK + b_rows * BK;
    uint32_t n = 0;
    int s = 0;
    uint32_t ph = 0, fills = 0;
    int drawn = static_cast<int>(blockIdx.x) / CTAS;       // the next tile (lane 0 of the first CTA)
    bool ok = true;
    for (;; ++n) {
      if (rank == 0 && lane == 0) {
        const int next = drawn < num_tiles ? drawn : -1;
        bars->tile[n % RING][0] = next;
        if (CTAS == 2)
          st_async_v4(mapa_u32(smem_u32(&bars->tile[n % RING]), 1), mapa_u32(smem_u32(&bars->tile_full[n % RING]), 1),
                      next, 0, 0, 0);
        mbar_arrive(&bars->tile_full[n % RING]);
      } else if (rank == 1 && lane == 0) {
        mbar_arrive_expect_tx(&bars->tile_full[n % RING], 16);
      }
      __syncwarp();
      int tile;
      if (!(ok = tile_at(n, tile)) || tile < 0) break;
      int tm, tn;
      coords(tile, tm, tn);
      const int m0 = tm * (BM * CTAS) + static_cast<int>(rank) * BM;
      const int n0 = tn * width + static_cast<int>(rank) * b_rows;
      for (int kb = 0; kb < k_blocks; kb += BLOCKS) {
        // the draw is on its way while the last stage of the tile is waited for
        if (rank == 0 && lane == 0 && kb + BLOCKS >= k_blocks) drawn = draws ? units + atomicAdd(counter, 1) : drawn + units;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->empty[s], ph ^ 1, p.status)))) break;
        if (elect_one()) {
          uint8_t* sa = smem + s * stage_bytes;
          const int have = min(BLOCKS, k_blocks - kb);
          if (rank == 0) mbar_arrive_expect_tx(&bars->full[s], CTAS * loaded * have);
#pragma unroll
          for (int i = 0; i < BLOCKS; ++i, sa += block_bytes) {
            if (i >= have) break;
            tma_load_2d_n<CTAS>(sa, &tmap_a, &bars->full[s], (kb + i) * BK, m0);
            tma_load_2d_n<CTAS>(sa + A_STAGE_BYTES, &tmap_b, &bars->full[s], (kb + i) * BK, n0);
          }
        }
        __syncwarp();
        ++fills;
        if (++s == stages) { s = 0; ph ^= 1; }
      }
      if (!ok) break;
    }
    grid_launch();
    if (draws && rank == 0 && lane == 0) {
      // Every unit draws until there is nothing left, so there are as many draws as tiles and the last one can rearm the counter.
      while (drawn < num_tiles) drawn = units + atomicAdd(counter, 1);        // after a wait that ran out
      if (drawn == units + num_tiles - 1) *counter = 0;
    }
    __syncwarp();
    if (ok) {
      for (int i = 0; i < stages && ok; ++i) {   // every stage handed back: no commit is on its way to these barriers
        ok = mbar_wait(&bars->empty[s], ph ^ 1, p.status);
        if (++s == stages) { s = 0; ph ^= 1; }
      }
    } else if (rank == 0) {
      for (int i = 0; i < stages; ++i) {         // let the copies already issued land
        if (fills <= static_cast<uint32_t>(i)) continue;
        mbar_wait(&bars->full[i], ((fills - 1 - i) / stages) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer (first CTA of a pair, for both)
    if (rank == 0) {
      const uint64_t da0 = umma_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t db0 = umma_desc_sw128(smem_u32(smem) + A_STAGE_BYTES, 16, 1024);
      int s = 0;
      uint32_t ph = 0, group = 0;
      bool ok = true;
      for (uint32_t n = 0; ok; ++n) {
        int tile;
        if (!(ok = tile_at(n, tile)) || tile < 0) break;
        const uint32_t acc = n & 1;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->acc_empty[acc], ((n >> 1) & 1) ^ 1, p.status)))) break;
        tc_fence_after();
        const uint32_t tmem_d = tmem_base + acc * MAX_WIDTH;
        for (int kb = 0; kb < k_blocks; kb += BLOCKS) {
          const uint32_t slot = group % SLOTS;
          if ((kb & 3) == 0 &&
              !(ok = __all_sync(0xffffffffu, mbar_wait(&bars->scale_full[slot], (group / SLOTS) & 1, p.status)))) break;
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->full[s], ph, p.status)))) break;
          tc_fence_after();
          const int end = min(kb + BLOCKS, k_blocks);
          const bool last = (end & 3) == 0 || end == k_blocks;          // of its group
          if (elect_one()) {
            const uint32_t scales = tmem_base + SLOT_COLUMN + slot * SLOT_COLUMNS;
            const uint32_t at = static_cast<uint32_t>(s * stage_bytes) >> 4;
            const uint32_t idesc = scaled_idesc(BM * CTAS, width, static_cast<uint32_t>(kb & 3));
#pragma unroll
            for (int i = 0; i < BLOCKS; ++i) {
              if (kb + i >= k_blocks) break;
              const uint32_t block = at + i * (static_cast<uint32_t>(block_bytes) >> 4);
#pragma unroll
              for (int k = 0; k < BK / UMMA_K; ++k)
                umma_scaled<CTAS>(tmem_d, da0 + block + k * (UMMA_K >> 4), db0 + block + k * (UMMA_K >> 4),
                                  idesc + i * NEXT_BYTE, scales, scales + 4, (kb > 0 || i > 0 || k > 0) ? 1u : 0u);
            }
            umma_commit_n<CTAS>(&bars->empty[s]);
            if (last) umma_commit_n<CTAS>(&bars->scale_empty[slot]);
            if (end == k_blocks) umma_commit_n<CTAS>(&bars->acc_full[acc]);
          }
          __syncwarp();
          if (last) ++group;
          if (++s == stages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp >= 4 + EPI_WARPS) {
    // ---------------------------------------------------------- scales
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t fills = 0;
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      int tile;
      if (!tile_at(n, tile) || tile < 0) break;
      int tm, tn;
      coords(tile, tm, tn);
      const int m0 = tm * (BM * CTAS) + static_cast<int>(rank) * BM + lane, n0 = tn * width + lane;
      for (int kb = 0; kb < k_blocks; kb += 4) {
        const uint32_t* wa = p.a_scales + static_cast<long long>(kb / 4) * p.a_pad;
        const uint32_t* wb = p.b_scales + static_cast<long long>(kb / 4) * p.b_pad;
        uint32_t a[4], b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = m0 + 32 * i < p.a_pad ? wa[m0 + 32 * i] : 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = 32 * i < width && n0 + 32 * i < p.b_pad ? wb[n0 + 32 * i] : 0u;
        const uint32_t slot = fills % SLOTS;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&bars->scale_empty[slot], ((fills / SLOTS) & 1) ^ 1, p.status)))) break;
        tc_fence_after();
        const uint32_t at = tmem_base + lanes + SLOT_COLUMN + slot * SLOT_COLUMNS;
        tmem_st_32x4(at, a);
        tmem_st_32x8(at + 4, b);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 2) mbar_arrive_cluster(mapa_u32(smem_u32(&bars->scale_full[slot]), 0));
          else mbar_arrive(&bars->scale_full[slot]);
        }
        ++fills;
      }
    }
    // every slot handed back: no commit is on its way to these barriers
    for (int i = 0; i < SLOTS && ok; ++i, ++fills)
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->scale_empty[fills % SLOTS], ((fills / SLOTS) & 1) ^ 1, p.status));
  } else if (warp >= 4) {
    // ---------------------------------------------------------- epilogue
    const int q = warp & 3;                     // TMEM lanes [32q, 32q + 32)
    const int half = (warp - 4) >> 2;           // odd or even 32-column chunks
    uint8_t* const stage = smem + BAR_OFF - (warp - 3) * C_STAGE_BYTES;
    for (uint32_t n = 0;; ++n) {
      int tile;
      if (!tile_at(n, tile) || tile < 0) break;
      const uint32_t acc = n & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&bars->acc_full[acc], (n >> 1) & 1, p.status))) break;
      int tm, tn;
      coords(tile, tm, tn);
      const int row0 = tm * (BM * CTAS) + static_cast<int>(rank) * BM + q * 32;
      const int n0 = tn * width;
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * MAX_WIDTH;
      constexpr int CHUNKS = F32 ? 1 : 2;       // chunks of 32 columns in flight: 2 KiB staged in bf16, 4 in fp32
      constexpr int BLOCK = C_STAGE_BYTES / CHUNKS;
#pragma unroll 1
      for (int c = half; c < width / 32; c += 2 * CHUNKS) {
        if (row0 >= p.M || n0 + c * 32 >= p.N) break;
        uint32_t r[CHUNKS][32];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j)
          if (j == 0 || c + 2 * j < width / 32) tmem_ld_32x32(taddr + (c + 2 * j) * 32, r[j]);
        tmem_ld_wait();
        if (lane == 0) bulk_wait_group_read<0>();      // the previous blocks have left the buffer
        __syncwarp();
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
          uint8_t* blk = stage + j * BLOCK;
          if (!F32) {
            // 64-byte rows, 16-byte chunks XOR-swizzled by the row pair
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const uint32_t* x = &r[j][8 * v];
              uint4 o;
              o.x = pack_bf16x2(__uint_as_float(x[0]), __uint_as_float(x[1]));
              o.y = pack_bf16x2(__uint_as_float(x[2]), __uint_as_float(x[3]));
              o.z = pack_bf16x2(__uint_as_float(x[4]), __uint_as_float(x[5]));
              o.w = pack_bf16x2(__uint_as_float(x[6]), __uint_as_float(x[7]));
              reinterpret_cast<uint4*>(blk + lane * 64)[v ^ ((lane >> 1) & 3)] = o;
            }
          } else {
            // 128-byte rows, 16-byte chunks XOR-swizzled by row
#pragma unroll
            for (int v = 0; v < 8; ++v)
              reinterpret_cast<uint4*>(blk + lane * 128)[v ^ (lane & 7)] =
                  make_uint4(r[j][4 * v], r[j][4 * v + 1], r[j][4 * v + 2], r[j][4 * v + 3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
#pragma unroll
          for (int j = 0; j < CHUNKS; ++j) {
            const int col0 = n0 + (c + 2 * j) * 32;
            if (j > 0 && (c + 2 * j >= width / 32 || col0 >= p.N)) continue;
            if (F32) tma_reduce_add_2d_bulk(&tmap_c, stage + j * BLOCK, col0, row0);
            else tma_store_2d_bulk(&tmap_c, stage + j * BLOCK, col0, row0);
          }
          bulk_commit_group();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) mbar_arrive_cluster(mapa_u32(smem_u32(&bars->acc_empty[acc]), 0));
        else mbar_arrive(&bars->acc_empty[acc]);
      }
    }
    if (lane == 0) bulk_wait_group<0>();         // staged blocks must leave before the CTA does
  }

  tc_fence_before();
  if (CTAS == 2) cluster_sync(); else __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_n<CTAS>(tmem_base, 512);
  }
}

template <int CTAS, bool F32, int BLOCKS>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Params& p, int num_sms, cudaStream_t stream) {
  auto kern = fp8_gemm_kernel<CTAS, F32, BLOCKS>;
  static std::atomic<uint64_t> configured{0};    // a bit for every device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return -2;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if ((configured.load(std::memory_order_relaxed) & bit) == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return -2;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  const int tiles = ((p.M + BM * CTAS - 1) / (BM * CTAS)) * ((p.N + p.width - 1) / p.width);
  const int units = num_sms / CTAS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CTAS * (tiles < units ? tiles : units)));
  cfg.blockDim = dim3(NUM_THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, ta, tb, tc, p) == cudaSuccess ? 0 : -3;
}

// Two k-blocks to a stage, and to a round of waiting and committing, where they leave room for four such stages (three for a
// CTA by itself).  A block costs the issuing warp as long as a narrow tile's MMAs take: 24 x 4096 x 14336 29.4 us by single blocks, 22.5
// by two (453 and 344 cycles a block of 64 columns); 1000 x 2048 x 8192 in pairs 18.9 and 16.0.
bool two_blocks(int ctas, int width) { return ctas == 2 ? width <= 128 : width <= 96; }

// Cycles of a launch by the model of the bf16 products (gemm_cost): an MMA of twice the elements per cycle on elements of half
// the size leaves the cycles per block of 128 bytes as they are there.  What the issue of a block takes is fitted to 14 shapes in
// all widths (M 16-4096, N 256-8192, K 256-14336), where the choice is 4 % behind the fastest on average.  A pair of which one CTA would
// have no rows is not considered: with weights from DRAM 24 x 4096 x 14336 takes 23.1 us as chosen and 23.3 in pairs of 64 columns,
// 128 x 4096 x 4096 9.5 and 10.0, but 100 x 2048 x 8192 14.4 and 13.0.
double cost(int M, int N, int K, bool f32, int ctas, int width, int num_sms) {
  const double k_blocks = (K + BK - 1) / BK;
  const long long tiles = static_cast<long long>((M + BM * ctas - 1) / (BM * ctas)) * ((N + width - 1) / width);
  const long long units = num_sms / ctas;
  const double rounds = static_cast<double>((tiles + units - 1) / units);
  const double fill = (std::min(M, BM) + width / ctas) * BK / 65.0;
  const double issue = ctas == 2 ? 250 : two_blocks(1, width) ? 295 + 0.8 * width : 430 + 0.4 * width;
  const double block = std::max({2.0 * width, fill, issue});
  const double epilogue = 2000 + (f32 ? 15 : 10) * width;
  return rounds * std::max(k_blocks * block, epilogue) + epilogue + (ctas == 2 ? 3600 : 2000);
}

// The counter of `stream`.  In rotation over the launches, two of them that run at once on two streams could have the same one, however
// many there are, when one has waited long enough; then tiles would be left out.  None while the stream is captured: the graph
// would keep it, and count in it beside later launches' CTAs when it is replayed on another stream.  None for the handle behind which
// every thread has another stream, and none for streams beyond the last counter.
int sched_slot(cudaStream_t stream) {
  static const bool fixed = [] {
    const char* env = getenv("PIPER_GEMM_STATIC_TILES");
    return env != nullptr && env[0] == '1';
  }();
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (fixed || stream == cudaStreamPerThread || cudaStreamIsCapturing(stream, &capture) != cudaSuccess ||
      capture != cudaStreamCaptureStatusNone || cudaStreamGetId(stream, &id) != cudaSuccess)
    return -1;
  static std::mutex mutex;
  static std::unordered_map<unsigned long long, int> slots;      // by the stream's id, which no later stream has again
  const std::lock_guard<std::mutex> lock(mutex);
  const auto known = slots.find(id);
  if (known != slots.end()) return known->second;
  if (slots.size() >= SCHED_SLOTS) return -1;
  return slots.emplace(id, static_cast<int>(slots.size())).first->second;
}

GemmShape shape_of(int M, int N, int K, bool f32, int num_sms) {
  GemmShape best = {1, MAX_WIDTH, 1};
  double least = 1e300;
  for (int ctas = 1; ctas <= (M > BM ? 2 : 1) && ctas <= num_sms; ++ctas)
    for (int width = MAX_WIDTH; width >= 32; width -= 32) {
      const double c = cost(M, N, K, f32, ctas, width, num_sms);
      if (c < least) {
        least = c;
        best = {ctas, width, 1};
      }
    }
  return best;
}

}  // namespace

int fp8_gemm_launch(const Fp8GemmArgs& g, int num_sms, cudaStream_t stream) {
  if (g.M <= 0 || g.N <= 0 || g.K <= 0) return 0;
  const GemmShape shape = shape_of(g.M, g.N, g.K, g.add_f32 != 0, num_sms);
  Params p;
  p.a_scales = g.a.scales;
  p.b_scales = g.b.scales;
  p.M = g.M;
  p.N = g.N;
  p.K = g.K;
  p.a_pad = static_cast<int>(fp8_scale_rows(g.M));
  p.b_pad = static_cast<int>(fp8_scale_rows(g.N));
  p.width = shape.width;
  // rows of A that do not exist need no room in the copy; what the stage holds there reaches no row that is stored
  p.a_rows = shape.ctas == 1 && g.M < BM ? (g.M + 7) / 8 * 8 : BM;
  const int b_rows = shape.width / shape.ctas;
  const int stage = A_STAGE_BYTES + b_rows * BK;
  const bool two = two_blocks(shape.ctas, shape.width);
  p.stages = std::min(MAX_STAGES, OPERAND_BYTES / (two ? 2 * stage : stage));
  const int tiles_m = (g.M + BM * shape.ctas - 1) / (BM * shape.ctas), tiles_n = (g.N + shape.width - 1) / shape.width;
  const bool n_fast = tiles_n < tiles_m;
  const long long fast_bytes = static_cast<long long>(n_fast ? g.N : g.M) * g.K;
  p.band = fast_bytes > (96ll << 20) ? 8 : (n_fast ? tiles_n : tiles_m);
  p.status = g.status;
  p.slot = sched_slot(stream);
  CUtensorMap ta, tb, tc;
  int rc = make_tmap_2d_u8(&ta, g.a.codes, g.K, g.M, g.a.ld, BK, p.a_rows);
  if (rc == 0) rc = make_tmap_2d_u8(&tb, g.b.codes, g.K, g.N, g.b.ld, BK, b_rows);
  if (rc == 0)
    rc = g.add_f32 ? make_tmap_c_f32(&tc, g.c, g.N, g.M, static_cast<uint64_t>(g.ldc) * 4)
                   : make_tmap_c_bf16(&tc, g.c, g.N, g.M, static_cast<uint64_t>(g.ldc) * 2);
  if (rc != 0) return rc;
  const int key = (shape.ctas == 2 ? 4 : 0) | (g.add_f32 ? 2 : 0) | (two ? 1 : 0);
  switch (key) {
    case 0: return launch<1, false, 1>(ta, tb, tc, p, num_sms, stream);
    case 1: return launch<1, false, 2>(ta, tb, tc, p, num_sms, stream);
    case 2: return launch<1, true, 1>(ta, tb, tc, p, num_sms, stream);
    case 3: return launch<1, true, 2>(ta, tb, tc, p, num_sms, stream);
    case 4: return launch<2, false, 1>(ta, tb, tc, p, num_sms, stream);
    case 5: return launch<2, false, 2>(ta, tb, tc, p, num_sms, stream);
    case 6: return launch<2, true, 1>(ta, tb, tc, p, num_sms, stream);
    default: return launch<2, true, 2>(ta, tb, tc, p, num_sms, stream);
  }
}

}  // namespace piper
