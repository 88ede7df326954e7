// Log-probabilities of given classes over rows of logits, with entropies and
// the top alternatives; the VJP of all three, and both in one call.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bc2n {

constexpr int LP_MAX_TOP = 32;

// One call's operands.  Null pointers leave an output unwritten or a
// cotangent zero.
struct LogProbs {
  int dtype = 0;  // of x and d: BC2N_F32, BC2N_F16, BC2N_BF16
  const void* x = nullptr;  // [rows][V], row stride ld elements
  int64_t ld = 0, rows = 0;
  int64_t total = 0;  // rows of the whole call, of which these may be a part
  int V = 0;
  const void* target = nullptr;  // [rows] i32 or (target64) i64; null: none
  int target64 = 0;
  int K = 0;  // alternatives
  float *logp = nullptr, *entropy = nullptr, *top_logp = nullptr;
  int32_t* top_index = nullptr;
  float* save = nullptr;  // [rows][4]: max, log of the sum, entropy, live (1 or 0)
  // backward
  const float *d_logp = nullptr, *d_entropy = nullptr, *d_top = nullptr;
  void* d = nullptr;  // [rows][V], row stride d_ld elements; may be x itself
  int64_t d_ld = 0;
};

// Bytes of the scratch that logprobs_fwd and logprobs_grad take (0: none).
size_t logprobs_work_bytes(int dtype, int64_t rows, int V, int K);
void logprobs_fwd(hipStream_t st, const LogProbs& a, void* work);
void logprobs_bwd(hipStream_t st, const LogProbs& a);
// forward without alternatives and backward of logp and entropy
void logprobs_grad(hipStream_t st, const LogProbs& a, void* work);

}  // namespace bc2n
