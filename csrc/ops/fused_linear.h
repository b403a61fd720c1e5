// Linear layer with bias, activation and residual behind its product, and with gradients (kernels/gated.cu, linear_few.cu, linear_pass.cu).
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <string>

namespace mccl {

// act(x w^T + bias) + residual; x [..., in], w [out, in].  activation: none, relu, silu, gelu, gelu_tanh.
at::Tensor fused_linear(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias, const std::string& activation,
                        const std::optional<at::Tensor>& residual);
// For tests: a 16-bit call without gradients whose kernels give every wait up after `wait_limit` cycles.
at::Tensor fused_linear_with_limit(const at::Tensor& x, const at::Tensor& w, int64_t wait_limit);

}  // namespace mccl
