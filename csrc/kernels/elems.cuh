// Runs of numbers between memory and fp32 registers, for kernels over fp32, fp16 and bf16 tensors.
#pragma once

#include "kernels/vec.cuh"

namespace mccl {
namespace kern {

// V numbers of a row: in chunks of 16 (or all 8) bytes where `vec` says that they are aligned to that, one by one and only the
// first n otherwise.
template <int kBytes> struct Chunk { using type = uint4; };
template <> struct Chunk<8> { using type = uint2; };

template <typename T, int V>
__device__ __forceinline__ void load_run(const T* p, int n, bool vec, float (&v)[V]) {
  constexpr int kBytes = V * sizeof(T) >= 16 ? 16 : V * sizeof(T), kPer = kBytes / sizeof(T);
  if constexpr (kBytes >= 8 && V % kPer == 0) {
    if (vec && n >= V) {
#pragma unroll
      for (int c = 0; c < V / kPer; ++c) {
        const auto raw = *reinterpret_cast<const typename Chunk<kBytes>::type*>(p + c * kPer);
        const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[c * kPer + i] = Traits<T>::load(x[i]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = i < n ? Traits<T>::load(p[i]) : 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void store_run(T* p, int n, bool vec, const float (&v)[V]) {
  constexpr int kBytes = V * sizeof(T) >= 16 ? 16 : V * sizeof(T), kPer = kBytes / sizeof(T);
  if constexpr (kBytes >= 8 && V % kPer == 0) {
    if (vec && n >= V) {
#pragma unroll
      for (int c = 0; c < V / kPer; ++c) {
        typename Chunk<kBytes>::type raw;
        T* x = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = Traits<T>::store(v[c * kPer + i]);
        *reinterpret_cast<typename Chunk<kBytes>::type*>(p + c * kPer) = raw;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = Traits<T>::store(v[i]);
}

// ---- 8-bit checkpoints ---------------------------------------------------------------------------------------
// A group's scale and what its numbers are multiplied with to become codes.  Two divisions a group, rounded to nearest, so that
// codes are the formula's in 32 bits, bit for bit.
constexpr int kGroup8 = 64;             // numbers with one scale
constexpr float kTiny8 = 0x1p-100f;     // below it 127 / most would overflow soon: such a group is kept as zeros
struct Scale8 {
  float scale, inverse;
};
__device__ __forceinline__ Scale8 scale8(float most) {
  if (!(most < INFINITY)) return {NAN, 0.f};  // an infinity or a NaN: the whole group comes back as NaN
  if (most < kTiny8) return {0.f, 0.f};
  return {__fdiv_rn(most, 127.f), __fdiv_rn(127.f, most)};
}
// Four codes, the first in the lowest byte.  `inverse` 0 (nothing to keep, or a NaN group): zeros, whatever x is.
__device__ __forceinline__ uint32_t codes8(float x0, float x1, float x2, float x3, float inverse) {
  const int a = __float2int_rn(x0 * inverse), b = __float2int_rn(x1 * inverse), c = __float2int_rn(x2 * inverse),
            d = __float2int_rn(x3 * inverse);
  const uint32_t w = (a & 0xFF) | (b & 0xFF) << 8 | (c & 0xFF) << 16 | static_cast<uint32_t>(d) << 24;
  return inverse == 0.f ? 0u : w;
}
__device__ __forceinline__ float value8(uint32_t word, int i, float scale) {
  return static_cast<float>(static_cast<int8_t>(word >> (8 * i))) * scale;
}
// The largest magnitude, a NaN where there is one (fmaxf drops it).
__device__ __forceinline__ float most8(float a, float x) {
  const float b = fabsf(x);
  return b != b ? b : (a != a ? a : fmaxf(a, b));
}

}  // namespace kern
}  // namespace mccl
