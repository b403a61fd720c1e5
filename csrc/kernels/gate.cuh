// The gate of a gated feed-forward block in fp32: act(z) = z s(z), s(z) = 1 / (1 + exp(-t)) with t = z (silu) or
// 2 sqrt(2/pi) (z + 0.044715 z^3) (gelu, tanh form).
#pragma once

namespace mccl {
namespace kern {

constexpr float kGelu = 1.5957691216057308f, kCubic = 0.044715f;  // 2 sqrt(2 / pi)

// silu within 6 roundings of 2^-24 of its size: the exponential's 4, the sum's and the quotient's.  gelu: t is itself rounded, five times
// 2^-24 of its size, which the exponential turns into as much relative to s where that is small: 5 |t| more.
__device__ __forceinline__ float gate_of(float z, bool silu) { return 1.f / (1.f + expf(-(silu ? z : kGelu * (z + kCubic * z * z * z)))); }

}  // namespace kern
}  // namespace mccl
