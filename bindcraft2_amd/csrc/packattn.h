// Attention of sequences packed one after another, with grouped heads, and
// its gradient.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "headnorm.h"

namespace bc2n {

constexpr int PA_MAX_WIDTH = 128;

struct PackedAttn {
  int dtype = 0;  // BC2N_F16, BC2N_BF16
  int causal = 0, fill = 0, sequences = 0;
  int heads = 0, kv_heads = 0, width = 0;
  int64_t q_tokens = 0, k_tokens = 0;
  float scale = 0;
  // [sequences + 1] first tokens; [sequences] lengths within them, or null
  const int32_t *q_off = nullptr, *k_off = nullptr, *q_len = nullptr, *k_len = nullptr;
  HeadView q, k, v, o;
  float* lse = nullptr;  // [heads][q_tokens]
  // backward
  HeadView d_o, dq, dk, dv;
};

size_t packattn_fwd_work_bytes(const PackedAttn& a);
size_t packattn_bwd_work_bytes(const PackedAttn& a);
void packattn_fwd(hipStream_t st, const PackedAttn& a, void* work);
void packattn_bwd(hipStream_t st, const PackedAttn& a, void* work);

}  // namespace bc2n
