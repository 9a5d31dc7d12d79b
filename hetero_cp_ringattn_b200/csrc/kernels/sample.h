// Host interface of the batched sampler.
#pragma once

#include <cuda_runtime.h>

namespace hcp {
namespace sampling {

// A per-row setting: an array when `ptr` is set, else one value for every row.
struct RowF {
  const float* ptr;
  float value;
};
struct RowI {
  const int* ptr;
  int value;
};

struct SampleArgs {
  const void* logits;  // [B] rows of V
  int bf16;            // 0: float32 logits, 1: bf16
  long row_stride;     // elements
  int B, V;
  const float* u;      // [B] uniform numbers in [0, 1)
  RowF temperature, top_p, min_p;
  RowI top_k;
  long long* token;    // [B]
  int num_sms;
};
const char* sample(const SampleArgs& a, cudaStream_t s);

}  // namespace sampling
}  // namespace hcp
