// AdamW step over tensors of several kinds (sm_100a): fp32 or bf16 parameters, moments in fp32 or in 8 bits, one launch.
//
//   p *= 1 - lr wd;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g;  p -= (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32, each operation rounded by itself, so that the result is the same bits wherever the formula is computed so.
//
// Moments in 8 bits: m as e4m3, v as e5m2, in units of a power of two that 256 numbers share, chosen so that the largest of them is at most
// 1.75 times the format's highest binade (448 and 57344).  A step moves v by a thousandth, far less than the format's steps: rounded to
// nearest it would never move.  So a number is rounded up as often as its place between two values asks for, by a hash of the element's number and
// the step: the mean over the steps is the fp32 moment's, and every replica of a model rounds alike.  What that leaves of noise in v, with steps
// of a seventh to a quarter and a thousand steps of memory, is about 0.3 of v, 0.15 of the step's size; in m, 0.09.  A v that is not zero stays
// at least the smallest code, for what divides by its root.  A group that holds an infinity or NaN is NaN as a whole from then on.
//
// bf16 parameters are the upper 16 bits of an fp32 value, rounded to nearest; `low` is what these leave of its bits, as a whole number.  A program that
// changes the parameter moves the value with it.  (fp32 copies of the parameters: 2 more bytes of traffic and of memory each, and they go stale.)
//
// 16.03 bytes a number (fp32 parameters), 14.03 (bf16), where fp32 moments have 28.  57 instructions a number (fp32 parameters), as pairs of numbers go
// through the packed fp32 instructions, 65 % of the issue slots, bf16 72 (78 without): 48 M numbers 143 us (5.6 TB/s), bf16 138 (5.1), with fp32 moments
// 206 (6.4); 96 M 269 (6.0), 271 (5.2) and 396 (6.6).  A warp has a group, so that what the group shares is two reductions; CTAs of two warps, ten to
// an SM (twelve, whose threads have fewer registers: 148, 139 and 207).  What is left is the start of each CTA, three reads behind each other,
// which the others have to fill.  (Without what is asked for ahead, or that in registers, which leaves half as many warps: 219; with
// the general root and quotient 235; CTAs of four warps 167; a third more room for what is asked for: 162.)
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/launch_count.h"
#include "kernels/optim_api.h"
#include "kernels/two.cuh"

namespace mccl {
namespace kern {

namespace {

constexpr int kThreads = 64, kWarps = kThreads / 32, kLane = 8;
constexpr int kShared = 7680;  // bytes a warp has for what it has asked for
static_assert(kMomentGroup == 32 * kLane, "a warp has a group");

// A hash of an element's number and the step, whose multipliers are digits of the roots of two and three.  Its lower 16 bits (the last round's
// exclusive or with the upper ones included) dither m, the upper ones v.  As words to add to the bits of a float that is shifted until its
// code is the upper byte: the dither below the code, and 64 above it, which is what the difference of the exponents' biases leaves of a byte.
struct Dither {
  uint32_t of_m, of_v;
  __device__ __forceinline__ Dither(uint32_t index, uint32_t step_word) {
    uint32_t h = (index ^ step_word) * 0x6A09E667u;
    h ^= h >> 15;
    h *= 0xBB67AE85u;
    of_v = __byte_perm(h, 0x40u, 0x4325);
    of_m = __byte_perm(h, 0x40u, 0x5105) ^ of_v;
  }
};

// The power of two that takes `most`, the bits of the largest number of a group, to at most 1.75 * 2^top: its exponent, biased.
__device__ __forceinline__ uint32_t power_of(uint32_t most, int top) {
  const int power = static_cast<int>((most + 0x1FFFFFu) >> 23) - top;
  return static_cast<uint32_t>(max(power, 127 - 120));
}
// a + b, with a one that the compiler does not know: of a product and a sum of pairs it makes one instruction, which rounds once, whatever is asked for.
__device__ __forceinline__ Two sum_of(Two a, Two b, Two one) { return fma_of(a, one, b); }
// Root and quotient, correctly rounded, of numbers far from either end of fp32's range, by Markstein's theorems (Computation of elementary
// functions on the IBM RISC System/6000 processor, 1990): Newton's iteration to a root or reciprocal within a rounding, then one step on the
// remainder, which a fused multiplication and addition gives exactly.  The theorem on quotients asks for a reciprocal that is correctly rounded itself,
// which the one step here may miss for a divisor beside a power of two (0x1.fffffe, 0x1.fffffa).  What that moves is some 2^-22 of a unit of the quotient,
// before it is rounded: it shows where a quotient is that near to the middle of two numbers.  All that are within 2^-20 are tested, and right.  No branch stands between one element's and the next one's, as
// there does in the general functions.  Signs are turned where that saves turning a factor's: -root(v), and a / -b.
__device__ __forceinline__ Two negative_root_of(Two v) {
  float a, b;
  v.apart(a, b);
  asm("rsqrt.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rsqrt.approx.ftz.f32 %0, %0;" : "+f"(b));
  const Two y(a, b), less_v = v * Two(-1.f), s = less_v * y, half = y * Two(0.5f), e = fma_of(s, half, Two(0.5f));
  const Two s1 = fma_of(s, e, s), half1 = fma_of(half, e, half);
  return fma_of(fma_of(s1, s1, less_v), half1, s1);
}
__device__ __forceinline__ Two quotient_of(Two a, Two less_b) {
  float b0, b1;
  less_b.apart(b0, b1);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b0) : "f"(-b0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b1) : "f"(-b1));
  const Two y0(b0, b1), y = fma_of(fma_of(less_b, y0, Two(1.f)), y0, y0), q = a * y;
  return fma_of(fma_of(less_b, q, a), y, q);
}
// Bits of the smallest and the largest number these are used for: 2^-60 and 2^60.
constexpr uint32_t kLeast = (127u - 60u) << 23, kMost = (127u + 60u) << 23;

// Values in units of their group's scale.
template <bool kFirst>
__device__ __forceinline__ void values_of(const uint32_t* codes, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw pair = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes[i / 2] >> (16 * (i % 2))), kFirst ? __NV_E4M3 : __NV_E5M2);
    const float2 f = __half22float2(__half2(pair));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// Of a lane's numbers, by magnitude, as bits.
struct Bounds {
  uint32_t most, least;
  __device__ __forceinline__ explicit Bounds(const float* x) {
    float a = x[0], b = x[0];
#pragma unroll
    for (int i = 1; i < kLane; i += 2) {  // (the last one twice)
      const float y = x[i], z = x[min(i + 1, kLane - 1)];
      asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(a) : "f"(y), "f"(z));
      asm("min.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(b) : "f"(y), "f"(z));
    }
    most = __float_as_uint(a);
    least = __float_as_uint(b);
  }
  __device__ __forceinline__ bool inside() const { return least >= kLeast && most <= kMost; }
};
// The upper bytes of four words as one word.
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
// A lane's 8 of a group's moments to codes, and the group's scale.  `dither`: one word a number.
//
// A positive float in units of the group becomes an 8-bit one with kDigits behind the point by adding the dither and cutting off the rest.
// Below the smallest normal number steps are even, as they are in the binade above it: there that number is added, and taken off as
// a code.  A warp whose numbers are all normal, as nearly all are, does without.
template <bool kFirst>
__device__ __forceinline__ void codes_of(const float* x, const Bounds& lane_bounds, const Dither* dither, float* scale, int lane, uint32_t* codes) {
  constexpr int kDigits = kFirst ? 3 : 2, kBias = kFirst ? 120 : 112;
  const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, lane_bounds.most), least = lane_bounds.least;
  const uint32_t power = power_of(most, kFirst ? 8 : 15);
  const bool finite = most < 0x7F800000u;
  const float inverse = __uint_as_float((254u - power) << 23), small = __uint_as_float((kBias + 1) << 23);
  if (lane == 0) *scale = finite ? __uint_as_float(power << 23) : __uint_as_float(0x7FC00000u);
  uint32_t word[kLane];
  if (__all_sync(0xFFFFFFFFu, __fmul_rn(__uint_as_float(least), inverse) >= small)) {
#pragma unroll
    for (int i = 0; i < kLane; i += 2) {  // (the shift drops the sign)
      float y[2];
      (Two(x[i], x[i + 1]) * Two(inverse)).apart(y[0], y[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) word[i + e] = (__float_as_uint(y[e]) << (1 + kDigits)) + (kFirst ? dither[i + e].of_m : dither[i + e].of_v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const float y = __fmul_rn(fabsf(x[i]), inverse);
      const bool low = y < small;
      const uint32_t sum = (__float_as_uint(low ? __fadd_rn(y, small) : y) << (1 + kDigits)) + (kFirst ? dither[i].of_m : dither[i].of_v);
      word[i] = low ? sum - (1u << (24 + kDigits)) : sum;
      if (!kFirst && y > 0.f) word[i] = max(word[i], 1u << 24);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    codes[w] = upper_bytes(word[4 * w], word[4 * w + 1], word[4 * w + 2], word[4 * w + 3]);
    if (kFirst)
      codes[w] |= 0x80808080u & upper_bytes(__float_as_uint(x[4 * w]), __float_as_uint(x[4 * w + 1]), __float_as_uint(x[4 * w + 2]), __float_as_uint(x[4 * w + 3]));
    if (!finite) codes[w] = 0u;
  }
}

// bf16 parameters and their lower bits, two a word, as fp32 values, and back.
__device__ __forceinline__ void join(const uint32_t* upper, const uint32_t* low, float* p) {
  float above[kLane];
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    above[i] = __uint_as_float(i % 2 ? upper[i / 2] & 0xFFFF0000u : upper[i / 2] << 16);
    uint32_t rest;  // with its sign in the upper half
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(rest) : "r"(low[i / 2]), "r"(i % 2 ? 0xBB32u : 0x9910u));
    p[i] = __uint_as_float(__float_as_uint(above[i]) + rest);
  }
  if (Bounds(above).least == 0u)  // a zero has nothing below it: its bits less one would be a NaN
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (above[i] == 0.f && __float_as_uint(p[i]) - __float_as_uint(above[i]) > 0x7FFFFFFFu) p[i] = above[i];
}
__device__ __forceinline__ void part(const float* p, uint32_t* upper, uint32_t* low) {
#pragma unroll
  for (int i = 0; i < kLane; i += 2) {
    const uint32_t a = __float_as_uint(p[i]), b = __float_as_uint(p[i + 1]);
    upper[i / 2] = __byte_perm(a + 0x8000u, b + 0x8000u, 0x7632);
    low[i / 2] = __byte_perm(a, b, 0x5410);  // what is above them takes no part in the difference's lower half
  }
  if (Bounds(p).most > 0x7F800000u)  // a NaN's bits may pass over into the sign
#pragma unroll
    for (int i = 0; i < kLane; ++i)
      if (isnan(p[i])) {
        const uint32_t kept = i % 2 ? 0xFFFFu : 0xFFFF0000u;
        upper[i / 2] = (upper[i / 2] & kept) | 0x7FC07FC0u & ~kept;
        low[i / 2] &= kept;
      }
}

// A tensor from the first number of a chunk on.
struct Chunk {
  void *param, *exp_avg, *exp_avg_sq;
  const void* grad;
  float *exp_avg_scale, *exp_avg_sq_scale;
  int16_t* low;
  int size;        // of the chunk
  uint32_t first;  // its first number's
  bool aligned;
  __device__ __forceinline__ Chunk(const AdamWTensor& t, const void* grad_of, int64_t begin, int chunk, int number_size, int moment_size) {
    param = static_cast<char*>(t.param) + begin * number_size;
    grad = static_cast<const char*>(grad_of) + begin * number_size;
    low = t.low + begin;
    exp_avg = static_cast<char*>(t.exp_avg) + begin * moment_size;
    exp_avg_sq = static_cast<char*>(t.exp_avg_sq) + begin * moment_size;
    exp_avg_scale = t.exp_avg_scale + begin / kMomentGroup;
    exp_avg_sq_scale = t.exp_avg_sq_scale + begin / kMomentGroup;
    size = static_cast<int>(min(static_cast<int64_t>(chunk), t.size - begin));
    first = static_cast<uint32_t>(begin);
    aligned = t.aligned && reinterpret_cast<uintptr_t>(grad_of) % 16 == 0;
  }
};

// Which 8 of a group's numbers are a lane's, so that its reads are runs of 16 bytes beside its neighbours': 8 in a row where no array has more
// than 16 bits a number, else two runs of 4.
template <bool kHalf, bool kEight>
struct Layout {
  static constexpr int kRuns = kHalf && kEight ? 1 : 2, kRun = kLane / kRuns, kApart = kMomentGroup / kRuns;
  static __device__ __forceinline__ int of(int lane) { return lane * kRun; }                       // its first number
  static __device__ __forceinline__ constexpr int number(int i) { return i / kRun * kApart + i % kRun; }  // its ith, from there
};

// What a lane reads of a group, as it comes from memory.  kHalf: a bf16 parameter; kEight: moments in 8 bits.
//
// Whole groups of aligned tensors are copied to shared memory kAhead of them ahead, each lane's to a place of its own, so that no lane waits
// for another one.
template <bool kHalf, bool kEight>
struct Raw {
  using L = Layout<kHalf, kEight>;
  static constexpr int kP = kHalf ? kLane / 2 : kLane, kM = kEight ? kLane / 4 : kLane;  // words
  static constexpr int kWords = kP * (kHalf ? 3 : 2) + 2 * kM;
  uint32_t p[kP], low[kHalf ? kP : 1], g[kP], m[kM], v[kM];
  float scale[2];

  // kN words in the array's runs, from the number `at` on, to the lane's places from `to` on; from these.  A run is 4, 8 or 16 bytes.
  template <int kN>
  static __device__ __forceinline__ void copy(const void* from, int at, uint32_t& to) {
    constexpr int kEach = kN / L::kRuns, kSize = 4 * kN / kLane;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r, to += 32 * 4 * kEach) {
      const char* f = static_cast<const char*>(from) + (at + r * L::kApart) * kSize;
      const uint32_t place = to + (threadIdx.x % 32) * (4 * kEach);
      if constexpr (kEach == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(place), "l"(f) : "memory");
      else if constexpr (kEach == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(place), "l"(f) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(place), "l"(f) : "memory");
    }
  }
  template <int kN>
  static __device__ __forceinline__ void take(uint32_t* to, uint32_t& from) {
    constexpr int kEach = kN / L::kRuns;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r, from += 32 * 4 * kEach, to += kEach) {
      const uint32_t place = from + (threadIdx.x % 32) * (4 * kEach);
      if constexpr (kEach == 4) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(to[0]), "=r"(to[1]), "=r"(to[2]), "=r"(to[3]) : "r"(place) : "memory");
      else if constexpr (kEach == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(to[0]), "=r"(to[1]) : "r"(place) : "memory");
      else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(to[0]) : "r"(place) : "memory");
    }
  }
  static __device__ __forceinline__ void ask(const Chunk& t, int at, uint32_t place) {
    copy<kP>(t.param, at, place);
    if constexpr (kHalf) copy<kP>(t.low, at, place);
    copy<kP>(t.grad, at, place);
    copy<kM>(t.exp_avg, at, place);
    copy<kM>(t.exp_avg_sq, at, place);
  }
  __device__ __forceinline__ void take(uint32_t place) {
    take<kP>(p, place);
    if constexpr (kHalf) take<kP>(low, place);
    take<kP>(g, place);
    take<kM>(m, place);
    take<kM>(v, place);
  }
  // One number at a time, and zeros behind the tensor.
  template <int kN>
  static __device__ __forceinline__ void singly(const void* from, int at, int size, uint32_t* to) {
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const int n = at + L::number(i);
      if constexpr (kN == kLane) {
        to[i] = n < size ? static_cast<const uint32_t*>(from)[n] : 0u;
      } else if constexpr (kN == kLane / 2) {
        const uint32_t x = n < size ? static_cast<const uint16_t*>(from)[n] : 0u;
        to[i / 2] = i % 2 ? to[i / 2] | x << 16 : x;
      } else {
        const uint32_t x = n < size ? static_cast<const uint8_t*>(from)[n] : 0u;
        to[i / 4] = i % 4 ? to[i / 4] | x << (8 * (i % 4)) : x;
      }
    }
  }
  __device__ __forceinline__ void singly(const Chunk& t, int at) {
    singly<kP>(t.param, at, t.size, p);
    if constexpr (kHalf) singly<kP>(t.low, at, t.size, low);
    singly<kP>(t.grad, at, t.size, g);
    singly<kM>(t.exp_avg, at, t.size, m);
    singly<kM>(t.exp_avg_sq, at, t.size, v);
  }
};

template <bool kHalf, bool kEight>
struct Group {
  using L = Layout<kHalf, kEight>;
  float p[kLane], m[kLane], v[kLane];

  __device__ __forceinline__ void update(const Raw<kHalf, kEight>& raw, const AdamWStep& h) {
    // (a power of two times a factor is no rounding of its own, nor is a code times that power: one product does for both)
    const float by_m = kEight ? __fmul_rn(raw.scale[0], h.beta1) : h.beta1, by_v = kEight ? __fmul_rn(raw.scale[1], h.beta2) : h.beta2;
    if constexpr (kEight) {
      values_of<true>(raw.m, m);
      values_of<false>(raw.v, v);
    }
    if constexpr (kHalf) join(raw.p, raw.low, p);
    const Two grad_scale(h.grad_scale), of_one(h.one_less_beta1), of_two(h.one_less_beta2), times_m(by_m), times_v(by_v), one(h.one);
#pragma unroll
    for (int i = 0; i < kLane; i += 2) {
      Two g;
      if constexpr (kHalf) {
        g = Two(__uint_as_float(raw.g[i / 2] << 16), __uint_as_float(raw.g[i / 2] & 0xFFFF0000u));
      } else {
        p[i] = __uint_as_float(raw.p[i]);
        p[i + 1] = __uint_as_float(raw.p[i + 1]);
        g = Two(__uint_as_float(raw.g[i]), __uint_as_float(raw.g[i + 1]));
      }
      if constexpr (!kEight) {
#pragma unroll
        for (int e = i; e < i + 2; ++e) {
          m[e] = __uint_as_float(raw.m[e]);
          v[e] = __uint_as_float(raw.v[e]);
        }
      }
      const Two d = g * grad_scale;
      sum_of(Two(m[i], m[i + 1]) * times_m, d * of_one, one).apart(m[i], m[i + 1]);
      sum_of(Two(v[i], v[i + 1]) * times_v, d * of_two * d, one).apart(v[i], v[i + 1]);
    }
    const Bounds of_m(m), of_v(v);
    if (h.ordinary && __all_sync(0xFFFFFFFFu, of_m.inside() && of_v.inside())) {
      const Two less_eps(-h.eps), inv_sqrt_bias2(h.inv_sqrt_bias2), decay(h.decay), less_step(-h.step_size);
#pragma unroll
      for (int i = 0; i < kLane; i += 2) {
        const Two less_below = sum_of(negative_root_of(Two(v[i], v[i + 1])) * inv_sqrt_bias2, less_eps, one);
        sum_of(Two(p[i], p[i + 1]) * decay, quotient_of(Two(m[i], m[i + 1]), less_below) * less_step, one).apart(p[i], p[i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const float below = __fadd_rn(__fmul_rn(__fsqrt_rn(v[i]), h.inv_sqrt_bias2), h.eps);
        p[i] = __fsub_rn(__fmul_rn(p[i], h.decay), __fmul_rn(__fdiv_rn(m[i], below), h.step_size));
      }
    }
  }

  // kN words in the array's runs, from the number `at` on.
  template <int kN>
  static __device__ __forceinline__ void put(void* to, int at, const uint32_t* from) {
    constexpr int kEach = kN / L::kRuns, kSize = 4 * kN / kLane;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r, from += kEach) {
      char* f = static_cast<char*>(to) + (at + r * L::kApart) * kSize;
      if constexpr (kEach == 4) *reinterpret_cast<uint4*>(f) = make_uint4(from[0], from[1], from[2], from[3]);
      else if constexpr (kEach == 2) *reinterpret_cast<uint2*>(f) = make_uint2(from[0], from[1]);
      else *reinterpret_cast<uint32_t*>(f) = from[0];
    }
  }
  template <int kN>
  static __device__ __forceinline__ void put_singly(void* to, int at, int size, const uint32_t* from) {
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const int n = at + L::number(i);
      if (n >= size) continue;
      if constexpr (kN == kLane) static_cast<uint32_t*>(to)[n] = from[i];
      else static_cast<uint16_t*>(to)[n] = static_cast<uint16_t>(from[i / 2] >> (16 * (i % 2)));
    }
  }
  // (codes are padded to whole groups)
  __device__ __forceinline__ void store(const Chunk& t, int at, int lane, bool whole, uint32_t step_word) const {
    if constexpr (kEight) {
      uint32_t codes[2];
      const uint32_t first = t.first + static_cast<uint32_t>(at);  // a multiple of a run
      const Dither dither[kLane] = {{first | L::number(0), step_word}, {first | L::number(1), step_word}, {first | L::number(2), step_word},
                                    {first | L::number(3), step_word}, {first | L::number(4), step_word}, {first | L::number(5), step_word},
                                    {first | L::number(6), step_word}, {first | L::number(7), step_word}};
      const int group = at / kMomentGroup;
      codes_of<true>(m, Bounds(m), dither, t.exp_avg_scale + group, lane, codes);
      put<2>(t.exp_avg, at, codes);
      codes_of<false>(v, Bounds(v), dither, t.exp_avg_sq_scale + group, lane, codes);
      put<2>(t.exp_avg_sq, at, codes);
    }
    constexpr int kP = Raw<kHalf, kEight>::kP;
    uint32_t words[kP], low[kP];
    if constexpr (kHalf) {
      part(p, words, low);
    } else {
#pragma unroll
      for (int i = 0; i < kP; ++i) words[i] = __float_as_uint(p[i]);
    }
    if (whole) {
      put<kP>(t.param, at, words);
      if constexpr (kHalf) put<kP>(t.low, at, low);
    } else {
      put_singly<kP>(t.param, at, t.size, words);
      if constexpr (kHalf) put_singly<kP>(t.low, at, t.size, low);
    }
    if constexpr (!kEight) {
      uint32_t first[kLane], second[kLane];
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        first[i] = __float_as_uint(m[i]);
        second[i] = __float_as_uint(v[i]);
      }
      if (whole) {
        put<kLane>(t.exp_avg, at, first);
        put<kLane>(t.exp_avg_sq, at, second);
      } else {
        put_singly<kLane>(t.exp_avg, at, t.size, first);
        put_singly<kLane>(t.exp_avg_sq, at, t.size, second);
      }
    }
  }
};

// A warp's groups of a chunk.
template <bool kHalf, bool kEight>
__device__ __forceinline__ void chunk_of(const AdamWTensor& tensor, const void* grad, const AdamWStep& h, int64_t begin, uint32_t shared) {
  using R = Raw<kHalf, kEight>;
  constexpr int kPlace = R::kWords * 128, kAhead = kShared / kPlace, kStep = kWarps * kMomentGroup;
  static_assert(kAhead >= 1, "one group at least");
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Chunk t(tensor, grad, begin, h.chunk, kHalf ? 2 : 4, kEight ? 1 : 4);
  // groups from `i` on: alike in a warp
  auto whole = [&](int i) { return t.aligned && i + kMomentGroup <= t.size; };
  auto ask = [&](int i, uint32_t place) {
    if (whole(i)) R::ask(t, i + Layout<kHalf, kEight>::of(lane), place);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int i = warp * kMomentGroup;
  const uint32_t first = shared + warp * kShared;
  uint32_t place = first;
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ask(i + k * kStep, first + k * kPlace);
  float scale[2] = {0.f, 0.f};
  auto scales = [&](int i) {
    if (kEight && i < t.size) {
      scale[0] = t.exp_avg_scale[i / kMomentGroup];
      scale[1] = t.exp_avg_sq_scale[i / kMomentGroup];
    }
  };
  scales(i);
#pragma unroll 1
  for (; i < t.size; i += kStep) {
    const int at = i + Layout<kHalf, kEight>::of(lane);
    R raw;
    raw.scale[0] = scale[0];
    raw.scale[1] = scale[1];
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    if (whole(i)) raw.take(place);
    else raw.singly(t, at);
    scales(i + kStep);
    Group<kHalf, kEight> group;
    group.update(raw, h);
    ask(i + kAhead * kStep, place);  // behind the last use of what was there
    place = place + kPlace == first + kAhead * kPlace ? first : place + kPlace;
    group.store(t, at, lane, whole(i), h.step_word);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

__global__ void __launch_bounds__(kThreads, 10) adamw_kinds_kernel(const AdamWTensor* __restrict__ tensors, const uint64_t* __restrict__ grads,
                                                               const int2* __restrict__ chunks, int num_chunks, const AdamWStep h) {
  __shared__ uint4 places[kWarps * kShared / 16];
  const uint32_t shared = static_cast<uint32_t>(__cvta_generic_to_shared(places));
  for (int c = blockIdx.x; c < num_chunks; c += gridDim.x) {
    const int2 place = chunks[c];
    const AdamWTensor t = tensors[place.x];
    const void* grad = reinterpret_cast<const void*>(grads[place.x]);
    const int64_t first = static_cast<int64_t>(place.y) * h.chunk;
    if (t.eight) {
      if (t.half) chunk_of<true, true>(t, grad, h, first, shared);
      else chunk_of<false, true>(t, grad, h, first, shared);
    } else {
      if (t.half) chunk_of<true, false>(t, grad, h, first, shared);
      else chunk_of<false, false>(t, grad, h, first, shared);
    }
  }
}

// For tests: what the step takes for a root of b and a quotient a / b, in either place beside another number; NaN where the places differ.
__global__ void root_quotient_kernel(const float* a, const float* b, float* root, float* quotient, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t j = n - 1 - i;
  float first, second, other;
  (negative_root_of(Two(b[i], b[j])) * Two(-1.f)).apart(first, other);
  (negative_root_of(Two(b[j], b[i])) * Two(-1.f)).apart(other, second);
  root[i] = __float_as_uint(first) == __float_as_uint(second) ? first : NAN;
  quotient_of(Two(a[i], a[j]), Two(-b[i], -b[j])).apart(first, other);
  quotient_of(Two(a[j], a[i]), Two(-b[j], -b[i])).apart(other, second);
  quotient[i] = __float_as_uint(first) == __float_as_uint(second) ? first : NAN;
}

}  // namespace

cudaError_t launch_root_quotient(const float* a, const float* b, float* root, float* quotient, int64_t n, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  note_launch();
  root_quotient_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(a, b, root, quotient, n);
  return cudaGetLastError();
}

cudaError_t launch_adamw_kinds(const AdamWTensor* tensors, const uint64_t* grads, const int2* chunks, int num_chunks, const AdamWStep& h, cudaStream_t s,
                               int max_ctas) {
  if (num_chunks <= 0) return cudaSuccess;
  note_launch();
  adamw_kinds_kernel<<<max_ctas > 0 && max_ctas < num_chunks ? max_ctas : num_chunks, kThreads, 0, s>>>(tensors, grads, chunks, num_chunks, h);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace mccl
