// Runs of numbers between memory and fp32 registers, for kernels over fp32, fp16 and bf16 tensors.
#pragma once

#include "kernels/vec.cuh"

namespace mccl {
namespace kern {

// Two numbers of 16 bits next to each other: one instruction, where two conversions and their joining are four.
template <typename T> __device__ __forceinline__ uint32_t store_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t store_pair<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t store_pair<__half>(float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
// V numbers as they lie in memory.
template <typename T, int V, typename Raw>
__device__ __forceinline__ Raw pack_run(const float* v) {
  Raw raw;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) reinterpret_cast<uint32_t*>(&raw)[i / 2] = store_pair<T>(v[i], v[i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) reinterpret_cast<T*>(&raw)[i] = Traits<T>::store(v[i]);
  }
  return raw;
}

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
        using Raw = typename Chunk<kBytes>::type;
        *reinterpret_cast<Raw*>(p + c * kPer) = pack_run<T, kPer, Raw>(&v[c * kPer]);
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
// Four codes, the first in the lowest byte: 1.5 2^23 and a number of at most 127 is a float whose lowest byte is that number,
// rounded to the nearest integer, halves to even.  (A conversion of each to an integer has a quarter of the additions' rate.)
// `inverse` 0 (nothing to keep, or a NaN group): zeros, whatever x is.
__device__ __forceinline__ uint32_t codes8(float x0, float x1, float x2, float x3, float inverse) {
  constexpr float kMagic = 12582912.f;
  const uint32_t a = __float_as_uint(__fadd_rn(__fmul_rn(x0, inverse), kMagic)), b = __float_as_uint(__fadd_rn(__fmul_rn(x1, inverse), kMagic)),
                 c = __float_as_uint(__fadd_rn(__fmul_rn(x2, inverse), kMagic)), d = __float_as_uint(__fadd_rn(__fmul_rn(x3, inverse), kMagic));
  const uint32_t w = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  return inverse == 0.f ? 0u : w;
}
// The values of four codes: a code and 128 in the lowest byte of 2^23 is that float, less 2^23 + 128 the code, exactly.  (A conversion
// has a quarter of an addition's rate.)
__device__ __forceinline__ void values8(uint32_t word, float scale, float* v) {
  const uint32_t w = word ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __fmul_rn(__fadd_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7540 + i)), -8388736.f), scale);
}
// The largest magnitude, as bits: those of a NaN are above those of all numbers.
__device__ __forceinline__ uint32_t most8(uint32_t most, float x) { return max(most, __float_as_uint(x) & 0x7FFFFFFFu); }

}  // namespace kern
}  // namespace mccl
