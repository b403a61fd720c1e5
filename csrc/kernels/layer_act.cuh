// Activations of a linear layer, as its kernels take them of fp32 sums, and their derivatives.
#pragma once

#include "kernels/gate.cuh"
#include "kernels/gated_api.h"

namespace mccl {
namespace kern {

// For results that are rounded to 16 bits.  Each is within 2^-18 of its size: exponentials and reciprocals by the instructions for them.
struct Act16 {
  static __device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  static __device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  // The logistic function of z, or of 2 sqrt(2 / pi) (z + 0.044715 z^3): s = 1 / (1 + 2^(z (c0 + c1 z^2))).  (Where the square overflows the
  // exponent does, to the right end.)
  static constexpr float kC0 = -1.4426950408889634f;
  static __device__ __forceinline__ float logistic(float z) { return reciprocal(1.f + exp2_of(kC0 * z)); }
  static __device__ __forceinline__ float cubic(float z, float square) { return reciprocal(1.f + exp2_of(z * fmaf(kC0 * kGelu * kCubic, square, kC0 * kGelu))); }
  // The normal distribution up to z, and its density times z.  The tail is t P(t) exp(-z^2 / 2) / 2 with t = 1 / (1 + |z| / sqrt(8)) and a polynomial
  // fitted to erfc(x) exp(x^2) / t by reweighted least squares, 2^-19.5 of its size off at most between x = 0 and 10.
  struct Normal {
    float share, slope;
  };
  static __device__ __forceinline__ Normal normal(float z) {
    const float a = fabsf(z), e = exp2_of(-0.7213475204444817f * fminf(a * a, 1e30f)), t = reciprocal(fmaf(a, 0.35355339059327373f, 1.f));
    float p = 0.0882045243f;
    p = fmaf(p, t, -0.35673875f);
    p = fmaf(p, t, 0.38922509f);
    p = fmaf(p, t, 0.0378904397f);
    p = fmaf(p, t, 0.281503786f);
    p = fmaf(p, t, 0.277582146f);
    p = fmaf(p, t, 0.282331411f);
    const float tail = 0.5f * t * p * e;
    return {z < 0.f ? tail : 1.f - tail, z * (0.3989422804014327f * e)};
  }
  template <LayerActivation kAct>
  static __device__ __forceinline__ float value(float z) {
    if constexpr (kAct == LayerActivation::kRelu) return z > 0.f || z != z ? z : 0.f;
    else if constexpr (kAct == LayerActivation::kSilu) return z * logistic(z);
    else if constexpr (kAct == LayerActivation::kGelu) return z * normal(z).share;
    else if constexpr (kAct == LayerActivation::kGeluTanh) return z * cubic(z, z * z);
    else return z;
  }
  template <LayerActivation kAct>
  static __device__ __forceinline__ float slope(float z) {
    if constexpr (kAct == LayerActivation::kRelu) {
      return z > 0.f ? 1.f : z != z ? z : 0.f;
    } else if constexpr (kAct == LayerActivation::kSilu) {
      const float s = logistic(z);
      return fmaf(z, fmaf(-s, s, s), s);
    } else if constexpr (kAct == LayerActivation::kGelu) {
      const Normal n = normal(z);
      return n.share + n.slope;
    } else if constexpr (kAct == LayerActivation::kGeluTanh) {
      const float square = fminf(z * z, 1e30f), s = cubic(z, square);
      return fmaf(z * fmaf(-s, s, s), fmaf(kGelu * 3.f * kCubic, square, kGelu), s);
    } else {
      return 1.f;
    }
  }
};
// For results in fp32: the functions of the CUDA library.
struct Act32 {
  template <LayerActivation kAct>
  static __device__ __forceinline__ float value(float z) {
    if constexpr (kAct == LayerActivation::kSilu || kAct == LayerActivation::kGeluTanh) return z * gate_of(z, kAct == LayerActivation::kSilu);
    else if constexpr (kAct == LayerActivation::kGelu) return z * normcdff(z);
    else return Act16::value<kAct>(z);
  }
  template <LayerActivation kAct>
  static __device__ __forceinline__ float slope(float z) {
    if constexpr (kAct == LayerActivation::kSilu || kAct == LayerActivation::kGeluTanh) {
      constexpr bool silu = kAct == LayerActivation::kSilu;
      const float s = gate_of(z, silu), t = s * (1.f - s);
      // (where the curve is flat the cubic's slope may be infinite)
      return t > 0.f ? s + z * t * (silu ? 1.f : kGelu * (1.f + 3.f * kCubic * z * z)) : s;
    } else if constexpr (kAct == LayerActivation::kGelu) {
      const float e = expf(-0.5f * z * z);
      return e > 0.f ? fmaf(z * 0.3989422804014327f, e, normcdff(z)) : normcdff(z);
    } else {
      return Act16::slope<kAct>(z);
    }
  }
};
// Calls `f` with the activation as a type.
template <LayerActivation kAct>
struct ActIs {
  static constexpr LayerActivation kValue = kAct;
};
#pragma nv_exec_check_disable
template <typename Call>
__host__ __device__ __forceinline__ auto with_activation(LayerActivation act, Call f) {
  switch (act) {
    case LayerActivation::kRelu: return f(ActIs<LayerActivation::kRelu>());
    case LayerActivation::kSilu: return f(ActIs<LayerActivation::kSilu>());
    case LayerActivation::kGelu: return f(ActIs<LayerActivation::kGelu>());
    case LayerActivation::kGeluTanh: return f(ActIs<LayerActivation::kGeluTanh>());
    default: return f(ActIs<LayerActivation::kNone>());
  }
}

}  // namespace kern
}  // namespace mccl
