// What kernels whose waits are bounded report to the host, and how the operators' CUDA calls are checked.
#pragma once

#include <ATen/ATen.h>
#include <cuda_runtime_api.h>

#include <algorithm>
#include <string>

#include "common/errors.h"

namespace mccl {

#define OPS_CK(expr)                                                         \
  do {                                                                       \
    cudaError_t _e = (expr);                                                 \
    if (_e != cudaSuccess) {                                                 \
      cudaGetLastError();                                                    \
      throw DeviceError(std::string(#expr) + ": " + cudaGetErrorString(_e)); \
    }                                                                        \
  } while (0)

// Words of mapped host memory, one per device, in which a kernel notes that one of its bounded waits ran out.
constexpr int kWaitDevices = 64;
inline uint32_t* wait_status(const at::Tensor& t) {
  static uint32_t* words = [] {
    void* p = nullptr;
    auto mode = cudaStreamCaptureModeRelaxed;  // the first call may be under capture
    OPS_CK(cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t e = cudaHostAlloc(&p, kWaitDevices * sizeof(uint32_t), cudaHostAllocMapped | cudaHostAllocPortable);
    OPS_CK(cudaThreadExchangeStreamCaptureMode(&mode));
    OPS_CK(e);
    std::fill_n(static_cast<uint32_t*>(p), kWaitDevices, 0u);
    return static_cast<uint32_t*>(p);
  }();
  return words + t.get_device() % kWaitDevices;
}
// Reports what a kernel has noted on the device, once.  What it gave up is NaN.
inline void check_waits(const at::Tensor& t) {
  uint32_t* word = wait_status(t);
  if (*static_cast<volatile uint32_t*>(word) != 0 && __atomic_exchange_n(word, 0u, __ATOMIC_RELAXED) != 0)
    throw DeviceError("a wait inside an earlier matrix product kernel ran out; what it should have written is NaN");
}

}  // namespace mccl
