// extern "C" entry point of the token draw (declared in include/dequant_b200.h):
// argument checks and the launch. Nothing here allocates device memory,
// synchronises or throws.
#include <cstdint>
#include <cuda_runtime.h>

#include "capi_checks.h"
#include "sampling.h"

extern "C" {

int dqg_sample_tokens(const void* logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                      const float* uniform, const dqg_sampling* params, int64_t* tokens, float* logprobs,
                      void* stream) {
  if (params == nullptr) return api_fail(DQG_ERR_INVALID, "params must not be null");
  if (dtype != DQG_FP16 && dtype != DQG_BF16 && dtype != DQG_FP32)
    return api_fail(DQG_ERR_INVALID, "dtype must be DQG_FP16, DQG_BF16 or DQG_FP32, got %d", dtype);
  if (rows < 0 || rows > (1 << 20)) return api_fail(DQG_ERR_INVALID, "rows=%lld out of range", (ll)rows);
  if (vocab < 1 || vocab > (1 << 18))
    return api_fail(DQG_ERR_UNSUPPORTED, "vocab must be in [1, 2^18], got %lld", (ll)vocab);
  if (rows == 0) return api_ok();
  if (rows > 1 && (row_stride < vocab || row_stride > (int64_t(1) << 38)))
    return api_fail(DQG_ERR_INVALID, "logits' row stride must be at least %lld, got %lld", (ll)vocab, (ll)row_stride);
  const void* ptrs[8] = {logits, uniform, tokens, logprobs, params->temperatures, params->top_ks, params->top_ps,
                         params->min_ps};
  const char* names[8] = {"logits", "uniform", "tokens", "logprobs", "temperatures", "top_ks", "top_ps", "min_ps"};
  const size_t align[8] = {dtype == DQG_FP32 ? size_t(4) : size_t(2), 4, 8, 4, 4, 4, 4, 4};
  int rc = DQG_OK;
  for (int i = 0; i < 8; ++i)
    if ((i < 4 || ptrs[i]) && (rc = check_ptr(ptrs[i], align[i], names[i])) != DQG_OK) return rc;
  int dev = 0, sms = 0;
  if ((rc = current(&dev, &sms)) != DQG_OK) return rc;
  dqg::SampleArgs a;
  a.logits = logits;
  a.row_stride = rows > 1 ? row_stride : vocab;
  a.uniform = uniform;
  a.temperatures = params->temperatures;
  a.top_ks = params->top_ks;
  a.top_ps = params->top_ps;
  a.min_ps = params->min_ps;
  a.tokens = tokens;
  a.logprobs = logprobs;
  a.temperature = params->temperature;
  a.top_k = params->top_k;
  a.top_p = params->top_p;
  a.min_p = params->min_p;
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.type = dtype;
  const cudaError_t e = dqg::launch_sample(a, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return api_cuda_fail(e, "sample_tokens launch");
  return api_ok();
}

}  // extern "C"
