// Host-side interface of the 8-bit products (fp8_quant.cu, fp8_gemm_sm100.cu).
//
// An operand is a matrix of e4m3 codes [rows, cols], cols along the contraction, rows `ld` bytes apart (a multiple of 16), with
// one power-of-two scale for every row and 128 columns.  Scales are exponents with a bias of 127 (255: NaN), four neighbouring ones
// of a row in one word: words [scale_groups(cols)][scale_rows(rows)], the row fastest.  A scale that a whole block of
// 128 x 128 shares stands in each of its rows.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piper {

constexpr int kFp8Group = 128;

inline long long fp8_scale_rows(long long rows) { return (rows + 127) / 128 * 128; }
inline long long fp8_scale_groups(long long cols) { return (cols + 4 * kFp8Group - 1) / (4 * kFp8Group); }

struct Fp8Out {
  uint8_t* codes;      // null: not wanted
  uint32_t* scales;
  long long ld;
};

// bf16 x [rows, cols], rows ldx elements apart (16-byte aligned vectors, cols % 16 == 0), as operand with the contraction along
// its columns (`plain`) and with the contraction along its rows (`turned`: codes [cols, rows]).  square: one scale
// for 128 x 128, the same in both.
int fp8_quantize(const void* x, long long rows, long long cols, long long ldx, int square, const Fp8Out& plain, const Fp8Out& turned,
                 cudaStream_t st);

// fp32 [rows, cols] of an operand.
int fp8_dequantize(const uint8_t* codes, const uint32_t* scales, long long ld, float* out, long long rows, long long cols, cudaStream_t st);

struct Fp8GemmArgs {
  const uint8_t* a;            // [M, K]
  const uint8_t* b;            // [N, K]
  const uint32_t* a_scales;
  const uint32_t* b_scales;
  void* c;                     // [M, N] bf16, or fp32 that is added to
  long long lda, ldb, ldc;
  int M, N, K;
  int add_f32;
  int* status;
};

// C = A B^T, or C += A B^T in fp32.
int fp8_gemm_launch(const Fp8GemmArgs& g, int num_sms, cudaStream_t st);

}  // namespace piper
