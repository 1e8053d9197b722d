// Host-side launchers of adamw.cu.  They enqueue on `st`, allocate nothing, and return 0 on success, -1 for
// more elements than a launch has chunks for and -3 for a launch error.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piper {

// 32 bits mixed by two multiplications, with the shifts and factors that C. Wellons published in 2018 (from a search for such mixers of
// little bias).
__host__ __device__ inline uint32_t mix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

constexpr int kMomentBlock = 256;      // elements that share a scale where moments have 8 bits
constexpr int kAdamwTensors = 80;      // tensors of one launch: their table travels with its arguments

// One tensor of an update.  Its moments (and its master copy) are the elements [at, at + n) of the state's buffers, with `at`
// a multiple of kMomentBlock.
struct AdamwTensor {
  float* weight;             // fp32: the parameter, or the master copy of a bf16 parameter
  void* param;               // bf16 parameter, or null
  const void* grad;
  long long n, at;
  float rate;                // lr / (1 - beta1^step)
  float root;                // 1 / sqrt(1 - beta2^step)
  unsigned seed;
  int grad_bf16;
};

struct AdamwTable {
  AdamwTensor t[kAdamwTensors];
  int first[kAdamwTensors + 1];        // chunk at which each tensor begins
  int count;
};

struct AdamwArgs {
  void* m;                   // uint8 codes (scales not null) or fp32
  void* v;
  float* m_scale;            // one per block, null where moments have 32 bits
  float* v_scale;
  float b1, b2, c1, c2;      // c1 = 1 - beta1, c2 = 1 - beta2
  float eps, keep;           // keep = 1 - lr * weight_decay
  int small_eps;             // the roots of numbers below the normal ones count beside eps
  float grad_scale;
};

// table.first and a.small_eps are filled in here.
int adamw_launch(AdamwTable& table, AdamwArgs a, int num_sms, cudaStream_t st);

// fp32 values of n codes of either moment (a multiple of kMomentBlock) with their scales.
int moments_decode(const void* m, const float* m_scale, const void* v, const float* v_scale, float* out_m, float* out_v, long long n,
                   cudaStream_t st);

}  // namespace piper
