// Host-side interface of the token draw (sampling.cu), called by
// capi_sampling.cu.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace dqg {

struct SampleArgs {
  const void* logits;  // [rows, vocab], rows row_stride elements apart
  int64_t row_stride;
  const float* uniform;        // [rows]
  const float* temperatures;   // [rows] or null: the value below
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  int64_t* tokens;  // [rows]
  float* logprobs;  // [rows]
  float temperature, top_p, min_p;
  int top_k;
  int rows, vocab;
  int type;  // DQG_FP16, DQG_BF16, DQG_FP32
};
cudaError_t launch_sample(const SampleArgs& a, int num_sms, cudaStream_t stream);

}  // namespace dqg
