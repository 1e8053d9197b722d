// Host-side interface of the 8-bit products (fp8_quant.cu, fp8_gemm_sm100.cu).
//
// An operand is a matrix of e4m3 codes [rows, cols], cols along the contraction, rows `ld` bytes apart (a multiple of 16), with
// one power-of-two scale for every row and 128 columns.  Scales are exponents with a bias of 127 (255: NaN), four neighbouring ones
// of a row in one word: words [scale_groups(cols)][scale_rows(rows)], the row fastest.  A scale that a whole block of
// 128 x 128 shares stands in each of its rows.  Codes and, behind them, words are one piece of memory.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piper {

constexpr int kFp8Group = 128;

inline long long fp8_scale_rows(long long rows) { return (rows + 127) / 128 * 128; }
inline long long fp8_scale_groups(long long cols) { return (cols + 4 * kFp8Group - 1) / (4 * kFp8Group); }

inline long long fp8_row_bytes(long long cols) { return (cols + 15) / 16 * 16; }
inline long long fp8_bytes(long long rows, long long cols) {
  return rows * fp8_row_bytes(cols) + 4 * fp8_scale_groups(cols) * fp8_scale_rows(rows);
}

struct Fp8Operand {
  uint8_t* codes;      // null: none
  uint32_t* scales;
  long long ld;

  // An operand [rows, cols] in fp8_bytes(rows, cols) of 16-byte aligned memory.
  static Fp8Operand at(void* memory, long long rows, long long cols) {
    if (memory == nullptr) return {nullptr, nullptr, 0};
    uint8_t* codes = static_cast<uint8_t*>(memory);
    const long long ld = fp8_row_bytes(cols);
    return {codes, reinterpret_cast<uint32_t*>(codes + rows * ld), ld};
  }
};

// bf16 x [rows, cols], rows ldx elements apart (16-byte aligned vectors, cols % 16 == 0), as operand with the contraction along
// its columns (`plain`) and with the contraction along its rows (`turned`: codes [cols, rows]).  square: one scale
// for 128 x 128, the same in both.
struct Fp8Rounding {
  const void* x;
  long long rows, cols, ldx;
  int square;
  Fp8Operand plain, turned;
};

// One or two matrices in one launch.
int fp8_quantize(const Fp8Rounding* what, int count, cudaStream_t st);

// fp32 [rows, cols] of an operand.
int fp8_dequantize(const Fp8Operand& a, float* out, long long rows, long long cols, cudaStream_t st);

struct Fp8GemmArgs {
  Fp8Operand a, b;             // [M, K], [N, K]
  void* c;                     // [M, N] bf16, or fp32 that is added to
  long long ldc;
  int M, N, K;
  int add_f32;
  int* status;
};

// C = A B^T, or C += A B^T in fp32.
int fp8_gemm_launch(const Fp8GemmArgs& g, int num_sms, cudaStream_t st);

}  // namespace piper
