// bf16 matrices to e4m3 codes with power-of-two scales, and back.
//
// The scale of a group is 2^e with the smallest e at which its largest magnitude is at most 448 * 2^e, 448 being the largest
// e4m3 number: 448 = 1.75 * 2^8, so e is the exponent of the largest magnitude minus 8, or minus 7 if its mantissa exceeds
// 1.75; bounded below by -127, the least a scale can say.  Dividing by a power of two is exact, so a code is the group's
// element rounded once, to the nearest code and ties to even, wherever it is computed.  A group with a NaN or an
// infinity has the scale NaN.
//
// What bounds it: memory.  A CTA takes 128 x 128 elements in one read and writes the codes along the rows, along the
// columns (which the gradient of the weights contracts over) or both: 2 bytes in, 1 or 2 out.  A thread holds eight rows of eight
// columns, so the eight codes of a column are one 8-byte word of the turned matrix; the words cross the CTA through shared memory
// to leave it in rows of 128 bytes.  4096 x 28672 along the rows 56 us (6.3 TB/s, floor 54), along both 85 (72).
#include "fp8.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "ptx.cuh"

namespace piper {
namespace {

constexpr int THREADS = 256;
constexpr int TILE = 128;

// Magnitudes are compared as the bits of bf16 numbers without their sign, two in a word; NaN and infinity are above all others.
__device__ __forceinline__ uint32_t magnitudes(uint32_t pair) { return pair & 0x7FFF7FFFu; }
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

// For a largest magnitude given by its bf16 bits (7 of mantissa): 8 more than the exponent, with its bias, of the scale.  31 carries
// into the exponent what is above 1.75.
__device__ __forceinline__ uint32_t scale_of(uint32_t most) { return max((most + 31u) >> 7, 8u); }
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) { return most >= 0x7F80u ? 255u : scale_of(most) - 8u; }
// 2^-e as a bf16 number, what elements are multiplied by.  e is 120 at most, and -127 at least, whose inverse is a normal number.
__device__ __forceinline__ uint32_t inverse_scale(uint32_t most) { return (262u - scale_of(most)) << 7; }

// Two bf16 products by powers of two, exact but for what is far below the smallest code.
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four codes of fp32 values, the first in the lowest byte.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

__device__ __forceinline__ float low_half(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_half(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }

struct Roundings {
  Fp8Rounding what[2];
  int tiles_x[2], tiles_y[2];
};

// Thread t: columns 8 (t % 16) to + 7, rows 8 (t / 16) to + 7 of a tile.  The tiles of the second matrix follow those of the first.
__global__ void __launch_bounds__(THREADS, 3)
fp8_quantize_kernel(const __grid_constant__ Roundings both) {
  grid_begin();
  const int first = both.tiles_x[0] * both.tiles_y[0];
  const int which = static_cast<int>(blockIdx.x) < first ? 0 : 1;
  const Fp8Rounding& r = both.what[which];
  const int tile = static_cast<int>(blockIdx.x) - which * first, tiles_x = both.tiles_x[which], tiles_y = both.tiles_y[which];
  const int tile_y = tile / tiles_x, tile_x = tile - tile_y * tiles_x;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(r.x);
  const long long rows = r.rows, cols = r.cols, ldx = r.ldx;
  const bool square = r.square != 0;
  const Fp8Operand &plain = r.plain, &turned = r.turned;
  __shared__ __align__(16) uint8_t turn[TILE * TILE];
  __shared__ __align__(16) uint32_t col_most[THREADS / 32][TILE / 2];      // two columns in a word
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
  const long long col0 = static_cast<long long>(tile_x) * TILE, row0 = static_cast<long long>(tile_y) * TILE;
  const long long c0 = col0 + 8 * l, r0 = row0 + 8 * g;
  uint4 v[8];
  const bool whole = col0 + TILE <= cols && row0 + TILE <= rows;
  {
    const __nv_bfloat16* p = x + r0 * ldx + c0;
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i, p += ldx) v[i] = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i, p += ldx)
        v[i] = c0 < cols && r0 + i < rows ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    }
  }

  uint32_t row_most[4];                          // of the thread's rows over all columns of the tile, two in a word
  uint32_t col_of[4] = {0, 0, 0, 0};             // of the thread's columns over all rows of the tile, likewise
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4& q = v[2 * i + h];
      m[h] = max2(max2(magnitudes(q.x), magnitudes(q.y)), max2(magnitudes(q.z), magnitudes(q.w)));
    }
    // even columns of both rows against odd ones of both
    row_most[i] = max2(__byte_perm(m[0], m[1], 0x5410), __byte_perm(m[0], m[1], 0x7632));
  }
  if (square) {
    uint32_t m = max2(max2(row_most[0], row_most[1]), max2(row_most[2], row_most[3]));
    m = __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
    if (lane == 0) col_most[0][warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) m = max(m, col_most[0][w]);
#pragma unroll
    for (int i = 0; i < 4; ++i) row_most[i] = col_of[i] = m | m << 16;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) row_most[i] = max2(row_most[i], __shfl_xor_sync(0xffffffffu, row_most[i], o));
    if (turned.codes != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t q[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) col_of[j] = max2(col_of[j], magnitudes(q[j]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) col_of[j] = max2(col_of[j], __shfl_xor_sync(0xffffffffu, col_of[j], 16));
      if (lane < 16) *reinterpret_cast<uint4*>(&col_most[warp][4 * l]) = make_uint4(col_of[0], col_of[1], col_of[2], col_of[3]);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        const uint4 o = *reinterpret_cast<const uint4*>(&col_most[w][4 * l]);
        col_of[0] = max2(col_of[0], o.x);
        col_of[1] = max2(col_of[1], o.y);
        col_of[2] = max2(col_of[2], o.z);
        col_of[3] = max2(col_of[3], o.w);
      }
    }
  }

  // The bytes of word (group of four, row); the last tile of a row fills the word.
  auto put_scale = [&](const Fp8Operand& o, long long block, long long blocks, long long row, long long pad, uint32_t byte) {
    uint8_t* word = reinterpret_cast<uint8_t*>(o.scales + block / 4 * pad + row);
    word[block & 3] = static_cast<uint8_t>(byte);
    if (block == blocks - 1)
      for (int b = static_cast<int>(block & 3) + 1; b < 4; ++b) word[b] = 0;
  };
  if (plain.codes != nullptr) {
    uint8_t* p = plain.codes + r0 * plain.ld + c0;
    uint32_t own = 0;                            // of row l: rows behind the end have words too, of zeros' scale
#pragma unroll
    for (int i = 0; i < 8; ++i, p += plain.ld) {
      const uint32_t most = i & 1 ? row_most[i / 2] >> 16 : row_most[i / 2] & 0xFFFFu;
      const uint32_t inv = inverse_scale(most) * 0x10001u;
      if (l == i) own = scale_byte(most);
      const uint32_t q[4] = {mul_bf16x2(v[i].x, inv), mul_bf16x2(v[i].y, inv), mul_bf16x2(v[i].z, inv), mul_bf16x2(v[i].w, inv)};
      const uint2 o = make_uint2(codes4(low_half(q[0]), high_half(q[0]), low_half(q[1]), high_half(q[1])),
                                 codes4(low_half(q[2]), high_half(q[2]), low_half(q[3]), high_half(q[3])));
      if (whole || (r0 + i < rows && c0 < cols)) *reinterpret_cast<uint2*>(p) = o;
    }
    if (l < 8) put_scale(plain, tile_x, tiles_x, r0 + l, static_cast<long long>(tiles_y) * TILE, own);
  }
  if (turned.codes != nullptr) {
    uint32_t own = 0;                            // of column 8 l + g
#pragma unroll
    for (int j = 0; j < 4; ++j) {                // two columns
      const uint32_t even = col_of[j] & 0xFFFFu, odd = col_of[j] >> 16;
      const uint32_t inv = inverse_scale(even) | inverse_scale(odd) << 16;
      if (g == 2 * j) own = scale_byte(even);
      if (g == 2 * j + 1) own = scale_byte(odd);
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = mul_bf16x2(j == 0 ? v[i].x : j == 1 ? v[i].y : j == 2 ? v[i].z : v[i].w, inv);
      // word g of column 8 l + 2 j, moved by l: the sixteen threads of a half warp meet sixteen pairs of banks
      uint8_t* const word = turn + (8 * l + 2 * j) * TILE + ((g ^ l) * 8);
      *reinterpret_cast<uint2*>(word) = make_uint2(codes4(low_half(q[0]), low_half(q[1]), low_half(q[2]), low_half(q[3])),
                                                   codes4(low_half(q[4]), low_half(q[5]), low_half(q[6]), low_half(q[7])));
      *reinterpret_cast<uint2*>(word + TILE) = make_uint2(codes4(high_half(q[0]), high_half(q[1]), high_half(q[2]), high_half(q[3])),
                                                          codes4(high_half(q[4]), high_half(q[5]), high_half(q[6]), high_half(q[7])));
    }
    if (g < 8) put_scale(turned, tile_y, tiles_y, c0 + g, static_cast<long long>(tiles_x) * TILE, own);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TILE * TILE / 16 / THREADS; ++k) {
      const int c = (threadIdx.x + k * THREADS) / 8, part = threadIdx.x & 7;       // column of x, 16 of its rows
      const int moved = c / 8;
      uint4 o = *reinterpret_cast<const uint4*>(turn + c * TILE + ((2 * part ^ moved) & ~1) * 8);
      if (moved & 1) o = make_uint4(o.z, o.w, o.x, o.y);
      // ld is rows rounded up to 16: what is behind the rows is zeros
      if (col0 + c < cols && row0 + 16 * part < turned.ld)
        *reinterpret_cast<uint4*>(turned.codes + (col0 + c) * turned.ld + row0 + 16 * part) = o;
    }
  }
}

__global__ void __launch_bounds__(THREADS)
fp8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint32_t* __restrict__ scales, long long ld, float* __restrict__ out,
                      long long rows, long long cols, long long pad) {
  grid_begin(codes, scales);
  const long long n = rows * cols;
  for (long long i = static_cast<long long>(blockIdx.x) * THREADS + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * THREADS) {
    const long long r = i / cols, c = i - r * cols, block = c / kFp8Group;
    const uint32_t byte = scales[block / 4 * pad + r] >> (8 * (block & 3)) & 255u;
    const __half_raw h = __nv_cvt_fp8_to_halfraw(codes[r * ld + c], __NV_E4M3);
    const float scale = byte == 255u ? __uint_as_float(0x7FC00000u) : byte == 0 ? __uint_as_float(1u << 22) : __uint_as_float(byte << 23);
    out[i] = __half2float(__half(h)) * scale;
  }
}

}  // namespace

int fp8_quantize(const Fp8Rounding* what, int count, cudaStream_t st) {
  Roundings both = {};
  long long tiles = 0;
  for (int i = 0; i < count && i < 2; ++i) {
    const Fp8Rounding& r = what[i];
    const long long x = (r.cols + TILE - 1) / TILE, y = (r.rows + TILE - 1) / TILE;
    if (r.cols % 16 != 0 || r.ldx % 8 != 0 || x > INT32_MAX / 2 || y > INT32_MAX / 2 || (tiles += x * y) > INT32_MAX / 2) return -1;
    both.what[i] = r;
    both.tiles_x[i] = static_cast<int>(x);
    both.tiles_y[i] = static_cast<int>(y);
  }
  if (tiles == 0) return 0;
  return launch_overlapped(fp8_quantize_kernel, static_cast<unsigned>(tiles), THREADS, 0, st, both) == cudaSuccess ? 0 : -3;
}

int fp8_dequantize(const Fp8Operand& a, float* out, long long rows, long long cols, cudaStream_t st) {
  if (rows == 0 || cols == 0) return 0;
  const long long want = (rows * cols + 8 * THREADS - 1) / (8 * THREADS);
  const dim3 grid(static_cast<unsigned>(want < 65536 ? want : 65536));
  return launch_overlapped(fp8_dequantize_kernel, grid, THREADS, 0, st, a.codes, a.scales, a.ld, out, rows, cols,
                           fp8_scale_rows(rows)) == cudaSuccess ? 0 : -3;
}

}  // namespace piper
