// Layer norm, with the sum before it and with gradients (kernels/norm.cu).
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <vector>

namespace mccl {

// y of x's type or `dtype`; with a residual also the sum of the two, in the residual's type, which is what is normed.
std::vector<at::Tensor> layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias, double eps,
                                   const std::optional<at::Tensor>& residual, std::optional<at::ScalarType> dtype);

}  // namespace mccl
