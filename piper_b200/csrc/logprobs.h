// Host-side launchers of logprobs.cu.  Both enqueue on `st`, allocate nothing, and return 0 on success, -1 for an
// unsupported shape and -3 for a launch error.
#pragma once
#include <cuda_runtime.h>

namespace piper {

constexpr int kMaxTopTokens = 32;
constexpr int kMaxVocabulary = 1 << 30;     // places in a row, and what is added to them, stay in 32 bits

// Logits [T, V] in bf16 or fp32 (f32 != 0), rows ld elements apart, any alignment of the type; z = logits / temperature.
struct LogprobArgs {
  const void* logits;
  const long long* tokens;      // [T]; one that is ignore_index or no id below V has log probability 0 and no gradient
  long long T, ld, ignore_index;
  int V, f32, top;              // top: alternatives per row, 0 to min(kMaxTopTokens, V)
  float inv_temperature;
};

// logprob, entropy [T]; top_logprob, top_id [T, top], by falling logits, equal ones by rising id; stats [T, 2] for the
// backward pass (largest logit, log2 of the sum of exp(z - largest z)).
int logprobs_fwd(const LogprobArgs& a, float* logprob, float* entropy, float* top_logprob, long long* top_id, float* stats,
                 int num_sms, cudaStream_t st);

// d [T, V], dense rows of the logits' type, from the gradients of the outputs (each null for none).
int logprobs_bwd(const LogprobArgs& a, const float* stats, const float* entropy, const long long* top_id,
                 const float* d_logprob, const float* d_entropy, const float* d_top, void* d, int num_sms, cudaStream_t st);

}  // namespace piper
