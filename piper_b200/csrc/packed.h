// Host-side launchers for packed batches: sequences of any lengths, one behind the other in T rows (pack.cu,
// attention_sm100.cu, policy.cu).  All enqueue on `st` and allocate nothing.  Return codes: 0 ok, -1 unsupported shape, -2 kernel
// attribute set-up failed, -3 launch error, >0 CUresult of a tensor-map encode.
#pragma once
#include <cuda_runtime.h>

namespace piper {

constexpr int kMaxPackedTokens = 1 << 21;      // two counters per 128 of them fit the shared memory of a CTA

// The table of a packed batch: [blocks + 1] rows of four ints.  Row 0: blocks in use, end of the last sequence, T, sequences
// that have rows (whose first blocks come last).  Then, for every block of 128 rows of a sequence, those with most blocks in front of
// them first: first row of the sequence, its rows, place of the block in the sequence, and 128 times the number of blocks of the
// sequences before (where lse and the like of it begin).
// own, unless null: neighbouring sequences that fit one block together count as one sequence, a group, with kGroup added to the
// fourth number, and of row i of a group own [blocks * 128][2] has the first and last row of its sequence in the group, at the place that
// lse begins at plus i.  Groups are formed within kGroupChunks parts of the sequences, of group_chunk(n) each.
// cu: n + 1 ints on the device, cu[0] == 0, rising, none above T; otherwise the table is empty and `status` set.
// scratch: 2 n ints with own, else unused.
constexpr int kGroup = 1, kGroupChunks = 32;
inline __host__ __device__ int group_chunk(int n) {
  const int c = (n + kGroupChunks - 1) / kGroupChunks;
  return c > 64 ? c : 64;
}
int pack_table(const int* cu, int n, int T, int blocks, int* table, unsigned char* own, int* scratch, int* status, cudaStream_t st);

struct PackedShape {
  const int* table;
  const unsigned char* own;    // null for a table without groups
  int T;
  long long blocks;            // that the table has memory for
  long long longest, work;     // about: blocks of the longest sequence, pairs of a query and a key block; choose launch shapes only
  int Hq, Hkv, hd;
};

// qkv [T, (Hq + 2 Hkv) hd] bf16 -> out [T, Hq hd] bf16, lse [Hq, 128 blocks] fp32 (natural log) and, unless null, rest
// [128 blocks, Hq hd]: what rounding has taken from out, for the backward pass, in an order of its own.
int attn_packed_fwd(const PackedShape& p, const void* qkv, void* out, float* lse, signed char* rest, float softmax_scale, int num_sms,
                    int* status, cudaStream_t st);

// d_qkv is overwritten whole.  rest may be null.  scratch: attn_packed_bwd_floats(); all 16-byte aligned.
long long attn_packed_bwd_floats(const PackedShape& p, int num_sms);
int attn_packed_bwd(const PackedShape& p, const void* qkv, const void* out, const signed char* rest, const void* d_out,
                    const float* lse, float* scratch, void* d_qkv, float softmax_scale, int num_sms, int* status, cudaStream_t st);

// Clipped policy loss.  logprob, old, adv, ref (or null) [T] fp32, mask [T] bytes or null; table null: one mean over all tokens.
struct PolicyArgs {
  const float *logprob, *old, *adv, *ref;
  const unsigned char* mask;
  const int* table;
  long long T, blocks;          // blocks: of the table, or of 128 tokens each
  double log_low, log_high;     // borders of logprob - old
  float low, high, kl_coef;
};

struct PolicyOut {
  float *loss, *kl, *clipped;   // the loss, the mean of e^u - 1 - u, the share of clipped tokens among those that count
  float* weight;                // 1 / (tokens that count); with a table 1 / (sequences that have some), and of a sequence at
                                // weight[1 + its first block] 1 / (tokens of it that count)
};

// scratch: 32 * blocks bytes, 8-byte aligned
int policy_fwd(const PolicyArgs& a, const PolicyOut& out, void* scratch, int num_sms, cudaStream_t st);
int policy_bwd(const PolicyArgs& a, const float* weight, const float* d_loss, float* d, int num_sms, cudaStream_t st);

// Balance loss of a router.  logits [T, E] bf16 or fp32 (f32 != 0), contiguous; idx [T, k]; mask [T] bytes or null.
constexpr int kMaxBalanceExperts = 256;
struct BalanceArgs {
  const void* logits;
  const int* idx;
  const unsigned char* mask;
  long long T;
  int E, k, f32;
  int* status;
};

// CTAs of balance_fwd, each of which has E + 1 numbers of 4 bytes twice in `scratch`.
int balance_ctas(long long T, int E, int num_sms);
// loss [1], counts [E], prob [E]; factor [E]: what the gradient of a probability is, up to that of the loss.
int balance_fwd(const BalanceArgs& a, float* loss, int* counts, float* prob, float* factor, void* scratch, int num_sms, cudaStream_t st);
int balance_bwd(const BalanceArgs& a, const float* factor, const float* d_loss, void* d, int num_sms, cudaStream_t st);

}  // namespace piper
