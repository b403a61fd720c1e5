// Gated feed-forward block with its gradients (kernels/gated.cu; fp32: kernels/gate_f32.cu between the products of ops/linear.h).
#pragma once

#include <ATen/ATen.h>

#include <string>

namespace mccl {

// (act(x w_gate^T) (x w_up^T)) w_down^T.  x [..., width], w_gate and w_up [hidden, width], w_down [width, hidden], all of one type.
// activation: "silu" or "gelu_tanh".  eight_bits: what the backward pass needs of x, g and u is kept in 8 bits.
at::Tensor gated_feed_forward(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, const at::Tensor& w_down,
                              const std::string& activation, bool eight_bits);
// For tests: a 16-bit forward pass whose kernels give every wait up after `wait_limit` cycles.
at::Tensor gated_with_limit(const at::Tensor& x, const at::Tensor& w_gate, const at::Tensor& w_up, const at::Tensor& w_down, int64_t wait_limit);

}  // namespace mccl
