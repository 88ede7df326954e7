// Root-mean-square norm of every head of queries and keys with the rotation
// by position, and its gradient.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bc2n {

// [tokens][heads][width], strides in elements, a head's elements contiguous
struct HeadView {
  const void* p = nullptr;
  int64_t st = 0, sh = 0;
};

struct HeadNorm {
  int dtype = 0, weight_dtype = 0;  // BC2N_F32, BC2N_F16, BC2N_BF16
  int64_t tokens = 0;
  int heads[2] = {0, 0};  // of queries and of keys
  int width = 0, rotated = 0, interleaved = 0;
  HeadView x[2], d[2], out[2];  // inputs, cotangents (backward), results
  const void* pos = nullptr;    // [tokens] i32 or (pos64) i64
  int pos64 = 0;
  const float* freq = nullptr;  // [rotated / 2]
  const void* weight[2] = {nullptr, nullptr};
  float eps = 0;
  float* d_weight[2] = {nullptr, nullptr};  // backward
};

// Elements of a rotated pair's vector: 0 if the widths have none.
int headnorm_vector(int dtype, int width, int rotated, int interleaved);
size_t headnorm_work_bytes(int64_t tokens, int width);
void headnorm_fwd(hipStream_t st, const HeadNorm& a);
void headnorm_bwd(hipStream_t st, const HeadNorm& a, void* work);

}  // namespace bc2n
