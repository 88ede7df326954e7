// A class a row of logits, drawn by given uniform numbers from the classes
// that temperature, top-k, top-p and min-p leave.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bc2n {

// A setting for all rows, or each row's own.
struct Setting {
  double v = 0;
  const float* row = nullptr;
};

struct Sample {
  int dtype = 0;            // of x: BC2N_F32, BC2N_F16, BC2N_BF16
  const void* x = nullptr;  // [rows][V], row stride ld elements
  int64_t ld = 0, rows = 0;
  int V = 0;
  const float* u = nullptr;  // [rows]
  Setting temperature, top_p, min_p;
  int64_t top_k = 0;
  const int32_t* top_k_row = nullptr;
  int32_t* index = nullptr;  // [rows]
  float* logp = nullptr;     // [rows], or null
};

void sample(hipStream_t st, const Sample& a);

}  // namespace bc2n
