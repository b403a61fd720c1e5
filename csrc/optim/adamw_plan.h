// AdamWPlan: device-resident launch plan of the fused multi-tensor AdamW kernel
// (kernels/adamw.cu): pointer tables of the parameters and their optimizer state, uploaded once,
// plus the table of gradient addresses, re-uploaded only when an address changed.  With extras it is the plan of the kernel
// for bf16 parameters and moments in 8 bits (kernels/adamw_kinds.cu).
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <cstring>
#include <vector>

#include "backend/tensor_checks.h"
#include "common/errors.h"
#include "kernels/optim_api.h"

namespace mccl {

#define MCCL_PLAN_CK(expr)                                                        \
  do {                                                                            \
    cudaError_t _e = (expr);                                                      \
    if (_e != cudaSuccess) {                                                      \
      cudaGetLastError();                                                         \
      throw DeviceError(std::string(#expr) + ": " + cudaGetErrorString(_e));      \
    }                                                                             \
  } while (0)

// A parameter's state beside its moments: scales where these are kept in 8 bits, the lower bits of a bf16 parameter.
struct AdamWExtra {
  at::Tensor exp_avg_scale, exp_avg_sq_scale, low;
};

class AdamWPlan {
 public:
  // Without extras: fp32 parameters and moments.
  AdamWPlan(std::vector<at::Tensor> params, std::vector<at::Tensor> exp_avg, std::vector<at::Tensor> exp_avg_sq, std::vector<AdamWExtra> extra = {})
      : params_(std::move(params)), m_(std::move(exp_avg)), v_(std::move(exp_avg_sq)), extra_(std::move(extra)) {
    MCCL_CHECK_TENSOR(!params_.empty() && params_.size() == m_.size() && params_.size() == v_.size() && (extra_.empty() || extra_.size() == params_.size()),
                      "AdamWPlan: list sizes differ");
    std::vector<int64_t> ptr_p, ptr_m, ptr_v, sizes;
    std::vector<int32_t> chunks;
    int64_t numbers = 0;
    bool eight = false;
    for (size_t i = 0; i < params_.size(); ++i) {
      check_tensors(i);
      numbers += params_[i].numel();
      eight = eight || m_[i].scalar_type() != at::kFloat;
    }
    chunk_ = extra_.empty() ? kern::kAdamWChunk : kern::adamw_kinds_chunk(numbers, eight);
    for (size_t i = 0; i < params_.size(); ++i) {
      ptr_p.push_back(reinterpret_cast<int64_t>(params_[i].data_ptr()));
      ptr_m.push_back(reinterpret_cast<int64_t>(m_[i].data_ptr()));
      ptr_v.push_back(reinterpret_cast<int64_t>(v_[i].data_ptr()));
      const int64_t n = params_[i].numel();
      sizes.push_back(n);
      for (int64_t c = 0; c * chunk_ < n; ++c) {
        chunks.push_back(static_cast<int32_t>(i));
        chunks.push_back(static_cast<int32_t>(c));
      }
    }
    auto dev = params_[0].device();
    auto up64 = [&](const std::vector<int64_t>& v) {
      return at::tensor(v, at::TensorOptions().dtype(at::kLong)).to(dev);
    };
    if (extra_.empty()) {
      d_p_ = up64(ptr_p);
      d_m_ = up64(ptr_m);
      d_v_ = up64(ptr_v);
      d_sizes_ = up64(sizes);
    } else {
      d_tensors_ = up64(tensor_table());
    }
    d_chunks_ = at::tensor(chunks, at::TensorOptions().dtype(at::kInt)).to(dev);
    num_chunks_ = static_cast<int>(chunks.size() / 2);
    grad_ptrs_.assign(params_.size(), 0);
    d_g_ = at::zeros({static_cast<int64_t>(params_.size())}, at::TensorOptions().dtype(at::kLong).device(dev));
  }

  // grads[i] may move between steps (zero_grad(set_to_none=True)); the pointer
  // table is re-uploaded only when an address changed.
  void step(const std::vector<at::Tensor>& grads, double lr, double beta1, double beta2, double eps,
            double weight_decay, int64_t step, double grad_scale) {
    bind_grads(grads);
    c10::cuda::CUDAGuard guard(params_[0].device());
    launch(at::cuda::getCurrentCUDAStream(), lr, beta1, beta2, eps, weight_decay, step, grad_scale);
  }

  // Points the plan at `grads` (uploads the pointer table only when an address changed).
  void bind_grads(const std::vector<at::Tensor>& grads) {
    MCCL_CHECK_TENSOR(grads.size() == params_.size(), "AdamWPlan.step: expected one gradient per parameter");
    bool changed = false;
    for (size_t i = 0; i < grads.size(); ++i) {
      const at::Tensor& g = grads[i];
      MCCL_CHECK_TENSOR(g.is_cuda() && g.device() == params_[i].device() && g.scalar_type() == params_[i].scalar_type() && g.is_contiguous() &&
                            g.numel() == params_[i].numel(),
                        "AdamWPlan.step: gradient " << i << " must be a contiguous tensor of the parameter's type and size, on its device");
      int64_t a = reinterpret_cast<int64_t>(g.data_ptr());
      if (a != grad_ptrs_[i]) {
        grad_ptrs_[i] = a;
        changed = true;
      }
    }
    if (changed) {
      c10::cuda::CUDAGuard guard(params_[0].device());
      at::Tensor host = at::tensor(grad_ptrs_, at::TensorOptions().dtype(at::kLong));
      d_g_.copy_(host);
    }
  }

  void launch(cudaStream_t stream, double lr, double beta1, double beta2, double eps, double weight_decay,
              int64_t step, double grad_scale, int max_ctas = 0) {
    const double bc1 = 1.0 - std::pow(beta1, static_cast<double>(step));
    const double bc2 = 1.0 - std::pow(beta2, static_cast<double>(step));
    if (!extra_.empty()) {
      // a replay would round with the same dither every time, and moments would drift
      cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
      MCCL_PLAN_CK(cudaStreamIsCapturing(stream, &capture));
      MCCL_CHECK_TENSOR(capture == cudaStreamCaptureStatusNone, "FusedAdamW: a step with moments in 8 bits or bfloat16 parameters cannot be captured, its number is the host's");
      kern::AdamWStep h;
      h.beta1 = static_cast<float>(beta1);
      h.one_less_beta1 = static_cast<float>(1.0 - beta1);
      h.beta2 = static_cast<float>(beta2);
      h.one_less_beta2 = static_cast<float>(1.0 - beta2);
      h.eps = static_cast<float>(eps);
      h.decay = static_cast<float>(1.0 - lr * weight_decay);
      h.step_size = static_cast<float>(lr / bc1);
      h.inv_sqrt_bias2 = static_cast<float>(1.0 / std::sqrt(bc2));
      h.grad_scale = static_cast<float>(grad_scale);
      h.one = 1.f;
      h.ordinary = h.eps >= 0.f && h.eps <= 0x1p20f && h.inv_sqrt_bias2 <= 0x1p20f;
      h.step_word = static_cast<uint32_t>(step) * 0x9E3779B9u;
      h.chunk = chunk_;
      MCCL_PLAN_CK(kern::launch_adamw_kinds(reinterpret_cast<const kern::AdamWTensor*>(d_tensors_.data_ptr<int64_t>()),
                                            reinterpret_cast<const uint64_t*>(d_g_.data_ptr<int64_t>()),
                                            reinterpret_cast<const int2*>(d_chunks_.data_ptr<int32_t>()), num_chunks_, h, stream, max_ctas));
      return;
    }
    kern::AdamWTable tab;
    tab.params = reinterpret_cast<const uint64_t*>(d_p_.data_ptr<int64_t>());
    tab.grads = reinterpret_cast<const uint64_t*>(d_g_.data_ptr<int64_t>());
    tab.exp_avg = reinterpret_cast<const uint64_t*>(d_m_.data_ptr<int64_t>());
    tab.exp_avg_sq = reinterpret_cast<const uint64_t*>(d_v_.data_ptr<int64_t>());
    tab.sizes = d_sizes_.data_ptr<int64_t>();
    tab.chunks = reinterpret_cast<const int2*>(d_chunks_.data_ptr<int32_t>());
    tab.num_chunks = num_chunks_;
    kern::AdamWHyper h;
    h.lr = static_cast<float>(lr);
    h.beta1 = static_cast<float>(beta1);
    h.beta2 = static_cast<float>(beta2);
    h.eps = static_cast<float>(eps);
    h.weight_decay = static_cast<float>(weight_decay);
    h.step_size = static_cast<float>(lr / bc1);
    h.inv_sqrt_bias2 = static_cast<float>(1.0 / std::sqrt(bc2));
    h.grad_scale = static_cast<float>(grad_scale);
    MCCL_PLAN_CK(kern::launch_adamw_multi(tab, h, stream, max_ctas));
  }
  int num_chunks() const { return num_chunks_; }
  const std::vector<at::Tensor>& params() const { return params_; }

 private:
  void check_tensors(size_t i) const {
    const at::Tensor& p = params_[i];
    auto fits = [&](const at::Tensor& t, at::ScalarType type, int64_t numel) {
      return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.scalar_type() == type && t.is_contiguous() && t.numel() == numel &&
             t.device() == params_[0].device();
    };
    if (extra_.empty()) {
      for (const at::Tensor* t : {&params_[i], &m_[i], &v_[i]})
        MCCL_CHECK_TENSOR(fits(*t, at::kFloat, p.numel()), "AdamWPlan: float32 contiguous CUDA tensors of one size and device only");
      return;
    }
    const bool half = p.scalar_type() == at::kBFloat16, eight = m_[i].scalar_type() == at::kFloat8_e4m3fn;
    MCCL_CHECK_TENSOR(fits(p, half ? at::kBFloat16 : at::kFloat, p.numel()), "AdamWPlan: contiguous float32 or bfloat16 CUDA parameters of one device only");
    MCCL_CHECK_TENSOR(half ? fits(extra_[i].low, at::kShort, p.numel()) : !extra_[i].low.defined(),
                      "AdamWPlan: bfloat16 parameters, and only these, have int16 lower bits of their size");
    if (eight) {
      const int64_t groups = (p.numel() + kern::kMomentGroup - 1) / kern::kMomentGroup;
      MCCL_CHECK_TENSOR(fits(m_[i], at::kFloat8_e4m3fn, groups * kern::kMomentGroup) && fits(v_[i], at::kFloat8_e5m2, groups * kern::kMomentGroup) &&
                            fits(extra_[i].exp_avg_scale, at::kFloat, groups) && fits(extra_[i].exp_avg_sq_scale, at::kFloat, groups) &&
                            (reinterpret_cast<uintptr_t>(m_[i].data_ptr()) | reinterpret_cast<uintptr_t>(v_[i].data_ptr())) % 8 == 0,
                        "AdamWPlan: moments in 8 bits are float8_e4m3fn and float8_e5m2, padded to whole groups of " << kern::kMomentGroup
                            << " from multiples of 8 bytes on, with a float32 scale for each");
    } else {
      // (scales are what the kernel takes moments of 8 bits by)
      MCCL_CHECK_TENSOR(fits(m_[i], at::kFloat, p.numel()) && fits(v_[i], at::kFloat, p.numel()) && !extra_[i].exp_avg_scale.defined() &&
                            !extra_[i].exp_avg_sq_scale.defined(),
                        "AdamWPlan: moments are float32 of the parameter's size, without scales");
    }
  }
  // Rows of kern::AdamWTensor.
  std::vector<int64_t> tensor_table() const {
    static_assert(sizeof(kern::AdamWTensor) % sizeof(int64_t) == 0, "rows of whole words");
    constexpr size_t kWords = sizeof(kern::AdamWTensor) / sizeof(int64_t);
    std::vector<int64_t> words(params_.size() * kWords);
    auto at = [](const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    for (size_t i = 0; i < params_.size(); ++i) {
      kern::AdamWTensor t{};
      t.param = params_[i].data_ptr();
      t.exp_avg = m_[i].data_ptr();
      t.exp_avg_sq = v_[i].data_ptr();
      t.exp_avg_scale = static_cast<float*>(at(extra_[i].exp_avg_scale));
      t.exp_avg_sq_scale = static_cast<float*>(at(extra_[i].exp_avg_sq_scale));
      t.low = static_cast<int16_t*>(at(extra_[i].low));
      t.size = params_[i].numel();
      t.half = t.low != nullptr;
      t.eight = t.exp_avg_scale != nullptr;
      uintptr_t all = reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.low);
      if (!t.eight) all |= reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq);
      t.aligned = all % 16 == 0;
      std::memcpy(words.data() + i * kWords, &t, sizeof(t));
    }
    return words;
  }

  std::vector<at::Tensor> params_, m_, v_;
  std::vector<AdamWExtra> extra_;
  std::vector<int64_t> grad_ptrs_;
  at::Tensor d_p_, d_g_, d_m_, d_v_, d_sizes_, d_chunks_, d_tensors_;
  int num_chunks_ = 0, chunk_ = 0;
};


}  // namespace mccl
