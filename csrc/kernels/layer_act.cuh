// Activations of a linear layer, as its kernels take them of fp32 sums, and their derivatives.
#pragma once

#include "kernels/gate.cuh"
#include "kernels/gated_api.h"
#include "kernels/two.cuh"

namespace mccl {
namespace kern {

// For products of 16-bit numbers.  Each is within 2^-18 of its size, a hundredth of the operands' own rounding in fp16, whether the result is rounded to 16
// bits or, with a residual in 32, is not: exponentials and reciprocals by the instructions for them.
// Of numbers (N: float) or of two side by side (Two), for which half as many instructions do.
struct Act16 {
  template <typename N>
  static __device__ __forceinline__ N exp2_of(N x) {
    return each_of(x, [](float x) {
      float y;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
      return y;
    });
  }
  template <typename N>
  static __device__ __forceinline__ N reciprocal(N x) {
    return each_of(x, [](float x) {
      float y;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
      return y;
    });
  }
  // The logistic function of z, or of 2 sqrt(2 / pi) (z + 0.044715 z^3): s = 1 / (1 + 2^(z (c0 + c1 z^2))).  (Where the square overflows the
  // exponent does, to the right end.)
  static constexpr float kC0 = -1.4426950408889634f;
  template <typename N>
  static __device__ __forceinline__ N logistic(N z) { return reciprocal(N(1.f) + exp2_of(N(kC0) * z)); }
  template <typename N>
  static __device__ __forceinline__ N cubic(N z, N square) {
    return reciprocal(N(1.f) + exp2_of(z * fma_of(N(kC0 * kGelu * kCubic), square, N(kC0 * kGelu))));
  }
  // The normal distribution up to z, and its density times z.  The tail is t P(t) exp(-z^2 / 2) / 2 with t = 1 / (1 + |z| / sqrt(8)) and a polynomial
  // fitted to erfc(x) exp(x^2) / t by reweighted least squares, 2^-19.5 of its size off at most between x = 0 and 10.
  template <typename N>
  struct Normal {
    N share, slope;
  };
  static __device__ __forceinline__ float share_of(float z, float tail) { return z < 0.f ? tail : 1.f - tail; }
  static __device__ __forceinline__ Two share_of(Two z, Two tail) {
    float a, b, s, t;
    z.apart(a, b);
    tail.apart(s, t);
    return Two(share_of(a, s), share_of(b, t));
  }
  template <typename N>
  static __device__ __forceinline__ Normal<N> normal(N z) {
    const N a = each_of(z, [](float z) { return fabsf(z); }), e = exp2_of(N(-0.7213475204444817f) * z * z);
    const N t = reciprocal(fma_of(a, N(0.35355339059327373f), N(1.f)));
    N p = N(0.0882045243f);
    p = fma_of(p, t, N(-0.35673875f));
    p = fma_of(p, t, N(0.38922509f));
    p = fma_of(p, t, N(0.0378904397f));
    p = fma_of(p, t, N(0.281503786f));
    p = fma_of(p, t, N(0.277582146f));
    p = fma_of(p, t, N(0.282331411f));
    return {share_of(z, N(0.5f) * t * p * e), z * (N(0.3989422804014327f) * e)};
  }
  template <LayerActivation kAct, typename N>
  static __device__ __forceinline__ N value(N z) {
    if constexpr (kAct == LayerActivation::kRelu) return each_of(z, [](float z) { return z > 0.f || z != z ? z : 0.f; });
    else if constexpr (kAct == LayerActivation::kSilu) return z * logistic(z);
    else if constexpr (kAct == LayerActivation::kGelu) return z * normal(z).share;
    else if constexpr (kAct == LayerActivation::kGeluTanh) return z * cubic(z, z * z);
    else return z;
  }
  template <LayerActivation kAct, typename N>
  static __device__ __forceinline__ N slope(N z) {
    static_assert(kAct != LayerActivation::kNone && kAct != LayerActivation::kRelu, "one and a choice");
    if constexpr (kAct == LayerActivation::kSilu) {
      const N s = logistic(z);
      return fma_of(z, fma_of(N(-1.f) * s, s, s), s);
    } else if constexpr (kAct == LayerActivation::kGelu) {
      const Normal<N> n = normal(z);
      return n.share + n.slope;
    } else {
      const N square = each_of(z * z, [](float x) { return fminf(x, 1e30f); }), s = cubic(z, square);
      return fma_of(z * fma_of(N(-1.f) * s, s, s), fma_of(N(kGelu * 3.f * kCubic), square, N(kGelu)), s);
    }
  }
  // Of kN numbers, each by its value.
  template <LayerActivation kAct, int kN>
  static __device__ __forceinline__ void values(float* z) {
    if constexpr (kAct != LayerActivation::kNone)
#pragma unroll
      for (int i = 0; i < kN; i += 2) value<kAct>(Two(z[i], z[i + 1])).apart(z[i], z[i + 1]);
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
    static_assert(kAct != LayerActivation::kNone && kAct != LayerActivation::kRelu, "one and a choice");
    if constexpr (kAct == LayerActivation::kSilu || kAct == LayerActivation::kGeluTanh) {
      constexpr bool silu = kAct == LayerActivation::kSilu;
      const float s = gate_of(z, silu), t = s * (1.f - s);
      // (where the curve is flat the cubic's slope may be infinite)
      return t > 0.f ? s + z * t * (silu ? 1.f : kGelu * (1.f + 3.f * kCubic * z * z)) : s;
    } else {
      const float e = expf(-0.5f * z * z);
      return e > 0.f ? fmaf(z * 0.3989422804014327f, e, normcdff(z)) : normcdff(z);
    }
  }
};
// The gradient of z from that of act(z).  relu's is a choice and no product: of what is infinite or NaN where z is not above zero nothing is left.
__device__ __forceinline__ float choice(float d, float z) { return z <= 0.f ? 0.f : d; }
__device__ __forceinline__ Two choice(Two d, Two z) {
  float a, b, x, y;
  d.apart(a, b);
  z.apart(x, y);
  return Two(choice(a, x), choice(b, y));
}
template <typename Act, LayerActivation kAct, typename N>
__device__ __forceinline__ N derived(N d, N z) {
  if constexpr (kAct == LayerActivation::kRelu) return choice(d, z);
  else return d * Act::template slope<kAct>(z);
}
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
