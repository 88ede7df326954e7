// Lists of gradients: their global 2-norm, their clipping, and the Adam
// update that takes the clipped gradients.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace bc2n {

// One tensor of a list; the operands a call does not have are null.
struct ListEntry {
  const void* g = nullptr;  // gradient
  void* g_out = nullptr;    // clipped gradient
  const void* p = nullptr;  // parameter, its first and second moments
  const float* m = nullptr;
  const float* v = nullptr;
  void* p_out = nullptr;
  float* m_out = nullptr;
  float* v_out = nullptr;
  int64_t n = 0;
  int32_t g_type = 0, p_type = 0;
  uint32_t chunk0 = 0;  // first chunk of the whole list's that is this tensor's
};

constexpr int LIST_INLINE = 32;  // tensors whose entries go with the launch

struct DeviceBlock {
  char* p = nullptr;
  size_t n = 0;
  int device = 0;
};

// A list as the kernels take it: cut into chunks of at most `chunk` elements
// of one tensor, a workgroup each.
class TensorList {
 public:
  // Checks the operands and, beyond LIST_INLINE tensors, uploads the entries.
  TensorList(std::vector<ListEntry> e, bool clips, bool adam);
  ~TensorList();
  TensorList(const TensorList&) = delete;
  TensorList& operator=(const TensorList&) = delete;

  size_t work_bytes() const;
  const bool clips;  // its gradients have outputs
  const bool adam;   // it has parameters and their moments

  // For a call captured into a graph: the graph may outlive the list, so the
  // list's table is never given to another.
  void keep_table() { kept_ = true; }

  static constexpr uint32_t MAGIC = 0x6c747362;
  uint32_t magic = MAGIC;

  std::vector<ListEntry> entries;  // the non-empty tensors
  int64_t total = 0, bytes = 0, chunk = 0;  // elements, of all operands, of a chunk
  uint32_t chunks = 0;
  ListEntry* dev = nullptr;        // device table (beyond LIST_INLINE)
  int32_t* dev_owner = nullptr;    // chunk -> entry

 private:
  DeviceBlock block_;
  bool kept_ = false;
};

struct AdamScalars {
  double lr = 0, beta1 = 0.9, beta2 = 0.999, eps = 1e-8, decay = 0;
  int64_t step = 1;
  double max_norm = 0;            // 0: not clipped
  const float* device = nullptr;  // {lr, step} on the device instead
};

// norm f32 [1]; max_norm > 0 scales the gradients into their outputs by
// max_norm / norm where the norm is not below it.
void grad_norm(hipStream_t st, const TensorList& l, float* norm, void* work);
void grad_clip(hipStream_t st, const TensorList& l, float max_norm, float* norm, void* work);
void adam_step(hipStream_t st, const TensorList& l, const AdamScalars& s, float* norm, void* work);

}  // namespace bc2n
