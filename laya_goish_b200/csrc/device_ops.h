// What the operators on caller-owned device buffers share (paging.cu,
// prefix_attn.cu, logprobs.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <exception>

#include "engine.h"
#include "laya_cuda.h"

namespace laya {

struct DeviceInfo {
  int device, sms;
  unsigned* status;  // the device's status word (LAYA_STATUS_* bits)
};
// The current device, which must be an sm_100 GPU; looked up once per device.
int device_info(DeviceInfo* out);
// Strides, alignment, sizes and type of a cache description; 0 or LAYA_E_INVALID.
int check_pages(const laya_kv_pages* c);
// laya_token_logprobs that reports in `status` (null: the device's word, which
// belongs to the callers of the operators).
int token_logprobs(uint32_t type, const void* logits, int64_t row_stride, int rows, int vocab, const int32_t* tokens,
                   int64_t token_stride, int n_tokens, int top, float* logprobs, float* entropy, float* lse,
                   int32_t* top_ids, float* top_logprobs, unsigned* status, cudaStream_t st);

// Runs an entry point's body; no C++ exception crosses the C boundary.
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      return fail(LAYA_E_NOMEM, e.what());
    } catch (...) {
      return LAYA_E_NOMEM;
    }
  } catch (...) {
    return LAYA_E_NOMEM;
  }
}

}  // namespace laya
