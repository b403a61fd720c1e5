// Activation checkpoints in 8 bits (kernels/pack8.cu).
#pragma once

#include <ATen/ATen.h>

#include <tuple>

namespace mccl {

// Codes [rows, pitch] (int8) and scales [rows, groups of 64] (fp32) of a CUDA tensor's rows along its last dimension.
std::tuple<at::Tensor, at::Tensor> pack8(const at::Tensor& x);
// The values, contiguous, of the given shape and type.
at::Tensor unpack8(const at::Tensor& codes, const at::Tensor& scales, at::IntArrayRef shape, at::ScalarType type);

}  // namespace mccl
