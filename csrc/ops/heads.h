// Norms and rotation of queries and keys, with gradients (kernels/heads.cu).
#pragma once

#include <ATen/ATen.h>

#include <tuple>

namespace mccl {


// q [batch, tokens, heads, dim], k [batch, tokens, kv heads, dim]; table [positions, 2, rotary / 2]; positions [tokens] or
// [batch, tokens], or none: 0, 1, ...
std::tuple<at::Tensor, at::Tensor> norm_rotate(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                               const at::Tensor& table, const c10::optional<at::Tensor>& positions, double eps, bool interleaved);
// The same of one projection [batch, tokens, (heads + 2 kv_heads) dim]; the third result is the view of its values.  One gradient.
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_rotate_packed(const at::Tensor& qkv, const at::Tensor& q_weight, const at::Tensor& k_weight,
                                                                  const at::Tensor& table, const c10::optional<at::Tensor>& positions,
                                                                  int64_t heads, int64_t kv_heads, double eps, bool interleaved);

}  // namespace mccl
