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
