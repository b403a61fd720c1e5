// What the operators of a decoder block share: their checks, types and error reports.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <string>

#include "kernels/pack8_api.h"
#include "ops/ordinary.h"
#include "ops/wait_status.h"

namespace mccl {

inline kern::Elem elem_of(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return kern::Elem::kF32;
    case at::kHalf: return kern::Elem::kF16;
    case at::kBFloat16: return kern::Elem::kBF16;
    default: throw TensorError(std::string(what) + ": float32, float16 or bfloat16 expected, got " + c10::toString(t.scalar_type()));
  }
}
// Whether a device is a B200, asked once.
inline bool device_fits(int device) {
  static std::atomic<uint64_t> fits{0};
  const uint64_t bit = 1ull << (device & 63);
  if (fits.load(std::memory_order_relaxed) & bit) return true;
  const auto* p = at::cuda::getDeviceProperties(static_cast<c10::DeviceIndex>(device));
  if (p->major != 10 || p->minor != 0) return false;
  if (device < 64) fits.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
// A tensor that the kernels may read: dense memory of a B200, no wrapper and no tangent that they would lose.
inline void check_block_tensor(const at::Tensor& t, const char* what) {
  MCCL_CHECK_T(TensorError, t.defined() && t.is_cuda() && t.layout() == at::kStrided, what << ": a dense CUDA tensor expected");
  MCCL_CHECK_T(TensorError, ordinary(t), what << ": tensor subclasses, transforms and forward-mode tangents are not supported");
  MCCL_CHECK_T(DeviceError, device_fits(t.get_device()), what << ": built for compute capability 10.0");
}
// A backward pass of kernels under a trace would leave its results in it as empty tensors.
inline void check_not_traced(const char* what) {
  const bool traced = c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
                      c10::impl::tls_local_dispatch_key_set().included_.has(c10::DispatchKey::PreDispatch);
  MCCL_CHECK_T(TensorError, !traced, what << ": the backward pass of a call outside of the trace cannot be traced");
}
// A tensor that was saved for the backward pass, as it comes back: a hook of the caller's may have laid it out anew, but may not have made
// another one of it, whose memory the kernels would run out of.
inline void check_saved(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device, const char* what) {
  check_block_tensor(t, what);
  MCCL_CHECK_T(TensorError, t.sizes() == sizes && t.scalar_type() == type && t.device() == device,
               what << ": a tensor saved for the backward pass came back as " << t.scalar_type() << " " << t.sizes() << " on " << t.device());
}
// Its numbers one behind the other from a multiple of 16 bytes on, as they were saved.
inline at::Tensor packed_again(const at::Tensor& t) {
  const at::Tensor r = t.contiguous();
  return reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 == 0 ? r : r.clone();
}
// `t` as rows along its last dimension: a view where its layout allows it, else a copy.
inline at::Tensor rows_of(const at::Tensor& t) {
  const int64_t cols = t.dim() ? t.size(-1) : 1;
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
  at::Tensor r = t.dim() == 2 ? t : t.reshape({rows, cols});
  if (r.numel() > 0 && (r.stride(1) != 1 && cols != 1)) r = r.contiguous();
  return r;
}
inline int64_t row_stride(const at::Tensor& r) { return r.size(0) <= 1 ? r.size(1) : r.stride(0); }

}  // namespace mccl
