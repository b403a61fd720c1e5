// Two fp32 numbers side by side, for the instructions that take both (sm_100a): each is rounded as by an instruction of its own, in one issue slot
// for the two.  (Of a product and a sum the compiler makes one instruction that rounds once, whatever rounding is asked for.)
#pragma once

#include <cstdint>

namespace mccl {
namespace kern {

struct Two {
  uint64_t bits;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ void apart(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two fma_of(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}
__device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
// `f` of each.
template <typename Call>
__device__ __forceinline__ Two each_of(Two x, Call f) {
  float a, b;
  x.apart(a, b);
  return Two(f(a), f(b));
}
template <typename Call>
__device__ __forceinline__ float each_of(float x, Call f) {
  return f(x);
}
// a += b, kN numbers.
template <int kN>
__device__ __forceinline__ void add_to(float* a, const float* b) {
  static_assert(kN % 2 == 0, "pairs");
#pragma unroll
  for (int i = 0; i < kN; i += 2) (Two(a[i], a[i + 1]) + Two(b[i], b[i + 1])).apart(a[i], a[i + 1]);
}

}  // namespace kern
}  // namespace mccl
