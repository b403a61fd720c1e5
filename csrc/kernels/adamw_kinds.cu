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
// Bound by memory: 16.03 bytes a number (fp32 parameters), 14.03 (bf16), where fp32 moments have 28.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/launch_count.h"
#include "kernels/optim_api.h"

namespace mccl {
namespace kern {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kLane = 8;
static_assert(kMomentGroup == 32 * kLane, "a warp has a group");

// Numbers of 16 bits for m (lower half) and v, from an element's number and the step; multipliers are the digits of square roots.
__device__ __forceinline__ uint32_t dither_of(uint32_t index, uint32_t step_word) {
  uint32_t h = (index ^ step_word) * 0x6A09E667u;  // sqrt(2)
  h ^= h >> 15;
  h *= 0xBB67AE85u;  // sqrt(3)
  return h ^ h >> 16;
}

// The power of two that takes `most`, the bits of the largest number of a group, to at most 1.75 * 2^top: its exponent, biased.
__device__ __forceinline__ uint32_t power_of(uint32_t most, int top) {
  const int power = static_cast<int>((most + 0x1FFFFFu) >> 23) - top;
  return static_cast<uint32_t>(max(power, 127 - 120));
}
// A positive float in units of its group as an 8-bit one with kDigits behind the point: truncated behind adding the dither to what is cut off.
// Below the smallest normal number steps are even, as they are in the binade above it: there it is added, and taken off as a code.
template <int kDigits>
__device__ __forceinline__ uint32_t code_of(float y, uint32_t dither) {
  constexpr int kBias = kDigits == 3 ? 120 : 112;
  const float small = __uint_as_float((kBias + 1) << 23);
  const bool low = y < small;
  const uint32_t bits = __float_as_uint(low ? __fadd_rn(y, small) : y) + (dither << (7 - kDigits));
  return (bits >> (23 - kDigits)) - ((low ? kBias + 1 : kBias) << kDigits);
}
template <bool kFirst>
__device__ __forceinline__ void values_of(uint2 codes, float scale, float* v) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw pair = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (16 * (i % 2))), kFirst ? __NV_E4M3 : __NV_E5M2);
    const float2 f = __half22float2(__half2(pair));
    v[2 * i] = __fmul_rn(f.x, scale);
    v[2 * i + 1] = __fmul_rn(f.y, scale);
  }
}
// A lane's 8 of a group's moments to codes, and the group's scale.  `dither`: one word a number.
template <bool kFirst>
__device__ __forceinline__ uint2 codes_of(const float* x, const uint32_t* dither, float* scale, int lane) {
  constexpr int kDigits = kFirst ? 3 : 2;
  uint32_t most = 0u;
#pragma unroll
  for (int i = 0; i < kLane; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  most = __reduce_max_sync(0xFFFFFFFFu, most);
  const uint32_t power = power_of(most, kFirst ? 8 : 15);
  const bool finite = most < 0x7F800000u;
  const float inverse = __uint_as_float((254u - power) << 23);
  if (lane == 0) *scale = finite ? __uint_as_float(power << 23) : __uint_as_float(0x7FC00000u);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const float y = __fmul_rn(fabsf(x[i]), inverse);
    uint32_t code = code_of<kDigits>(y, kFirst ? dither[i] & 0xFFFFu : dither[i] >> 16);
    if (kFirst) code |= __float_as_uint(x[i]) >> 31 << 7;
    else if (y > 0.f) code = max(code, 1u);
    w[i / 4] |= code << (8 * (i % 4));
  }
  return finite ? make_uint2(w[0], w[1]) : make_uint2(0u, 0u);
}

__device__ __forceinline__ float joined(uint32_t upper, uint32_t low) {  // 16 bits each
  const int rest = static_cast<int16_t>(low);
  // (a zero has nothing below it: its bits less one would be a NaN)
  return __uint_as_float((upper << 16) + ((upper & 0x7FFFu) == 0u && rest < 0 ? 0 : rest));
}
__device__ __forceinline__ void parted(float p, uint32_t& upper, uint32_t& low) {
  const uint32_t bits = __float_as_uint(p);
  const bool nan = (bits & 0x7FFFFFFFu) > 0x7F800000u;
  upper = nan ? 0x7FC0u : (bits + 0x8000u) >> 16;
  low = nan ? 0u : (bits - (upper << 16)) & 0xFFFFu;
}

// kHalf: a bf16 parameter; kEight: moments in 8 bits.
template <bool kHalf, bool kEight>
struct Group {
  float p[kLane], g[kLane], m[kLane], v[kLane];

  __device__ __forceinline__ void load(const AdamWTensor& t, const void* grad, int64_t at, int lane, bool whole) {
    if (whole) {
      if constexpr (kHalf) {
        const uint4 up = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t.param) + at), lo = *reinterpret_cast<const uint4*>(t.low + at),
                    gr = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(grad) + at));
        const uint32_t u[4] = {up.x, up.y, up.z, up.w}, l[4] = {lo.x, lo.y, lo.z, lo.w}, d[4] = {gr.x, gr.y, gr.z, gr.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[2 * i] = joined(u[i] & 0xFFFFu, l[i] & 0xFFFFu);
          p[2 * i + 1] = joined(u[i] >> 16, l[i] >> 16);
          g[2 * i] = __uint_as_float(d[i] << 16);
          g[2 * i + 1] = __uint_as_float(d[i] & 0xFFFF0000u);
        }
      } else {
        vector(static_cast<const float*>(t.param) + at, p, false);
        vector(static_cast<const float*>(grad) + at, g, true);
      }
      if constexpr (!kEight) {
        vector(static_cast<const float*>(t.exp_avg) + at, m, false);
        vector(static_cast<const float*>(t.exp_avg_sq) + at, v, false);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        const bool there = at + i < t.size;
        p[i] = g[i] = 0.f;
        if constexpr (!kEight) m[i] = v[i] = 0.f;
        if (!there) continue;
        if constexpr (kHalf) {
          p[i] = joined(static_cast<const uint16_t*>(t.param)[at + i], static_cast<uint16_t>(t.low[at + i]));
          g[i] = __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(grad)[at + i]) << 16);
        } else {
          p[i] = static_cast<const float*>(t.param)[at + i];
          g[i] = static_cast<const float*>(grad)[at + i];
        }
        if constexpr (!kEight) {
          m[i] = static_cast<const float*>(t.exp_avg)[at + i];
          v[i] = static_cast<const float*>(t.exp_avg_sq)[at + i];
        }
      }
    }
    if constexpr (kEight) {
      const int64_t group = at / kMomentGroup;  // codes are padded to whole groups
      values_of<true>(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.exp_avg) + at), t.exp_avg_scale[group], m);
      values_of<false>(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.exp_avg_sq) + at), t.exp_avg_sq_scale[group], v);
      if (!whole)
#pragma unroll
        for (int i = 0; i < kLane; ++i)
          if (at + i >= t.size) m[i] = v[i] = 0.f;
    }
  }
  static __device__ __forceinline__ void vector(const float* from, float* to, bool once) {
    const float4* f = reinterpret_cast<const float4*>(from);
    const float4 a = once ? __ldcs(f) : f[0], b = once ? __ldcs(f + 1) : f[1];
    to[0] = a.x, to[1] = a.y, to[2] = a.z, to[3] = a.w, to[4] = b.x, to[5] = b.y, to[6] = b.z, to[7] = b.w;
  }

  __device__ __forceinline__ void update(const AdamWStep& h) {
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const float d = __fmul_rn(g[i], h.grad_scale);
      m[i] = __fadd_rn(__fmul_rn(m[i], h.beta1), __fmul_rn(d, h.one_less_beta1));
      v[i] = __fadd_rn(__fmul_rn(v[i], h.beta2), __fmul_rn(__fmul_rn(d, h.one_less_beta2), d));
      const float below = __fadd_rn(__fmul_rn(__fsqrt_rn(v[i]), h.inv_sqrt_bias2), h.eps);
      p[i] = __fsub_rn(__fmul_rn(p[i], h.decay), __fmul_rn(__fdiv_rn(m[i], below), h.step_size));
    }
  }

  __device__ __forceinline__ void store(const AdamWTensor& t, int64_t at, int lane, bool whole, uint32_t step_word) const {
    if constexpr (kEight) {
      uint32_t dither[kLane];
#pragma unroll
      for (int i = 0; i < kLane; ++i) dither[i] = dither_of(static_cast<uint32_t>(at) + i, step_word);
      const int64_t group = at / kMomentGroup;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(t.exp_avg) + at) = codes_of<true>(m, dither, t.exp_avg_scale + group, lane);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(t.exp_avg_sq) + at) = codes_of<false>(v, dither, t.exp_avg_sq_scale + group, lane);
    }
    uint32_t upper[kLane], low[kLane];
    if constexpr (kHalf)
#pragma unroll
      for (int i = 0; i < kLane; ++i) parted(p[i], upper[i], low[i]);
    if (whole) {
      if constexpr (kHalf) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(t.param) + at) =
            make_uint4(upper[0] | upper[1] << 16, upper[2] | upper[3] << 16, upper[4] | upper[5] << 16, upper[6] | upper[7] << 16);
        *reinterpret_cast<uint4*>(t.low + at) = make_uint4(low[0] | low[1] << 16, low[2] | low[3] << 16, low[4] | low[5] << 16, low[6] | low[7] << 16);
      } else {
        put(static_cast<float*>(t.param) + at, p);
      }
      if constexpr (!kEight) {
        put(static_cast<float*>(t.exp_avg) + at, m);
        put(static_cast<float*>(t.exp_avg_sq) + at, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLane; ++i) {
        if (at + i >= t.size) continue;
        if constexpr (kHalf) {
          static_cast<uint16_t*>(t.param)[at + i] = static_cast<uint16_t>(upper[i]);
          t.low[at + i] = static_cast<int16_t>(low[i]);
        } else {
          static_cast<float*>(t.param)[at + i] = p[i];
        }
        if constexpr (!kEight) {
          static_cast<float*>(t.exp_avg)[at + i] = m[i];
          static_cast<float*>(t.exp_avg_sq)[at + i] = v[i];
        }
      }
    }
  }
  static __device__ __forceinline__ void put(float* to, const float* from) {
    reinterpret_cast<float4*>(to)[0] = make_float4(from[0], from[1], from[2], from[3]);
    reinterpret_cast<float4*>(to)[1] = make_float4(from[4], from[5], from[6], from[7]);
  }
};

template <bool kHalf, bool kEight>
__device__ __forceinline__ void chunk_of(const AdamWTensor& t, const void* grad, const AdamWStep& h, int chunk) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t first = static_cast<int64_t>(chunk) * kAdamWChunk;
  const bool aligned = t.aligned && reinterpret_cast<uintptr_t>(grad) % 16 == 0;
#pragma unroll 1
  for (int i = warp; i < kAdamWChunk / kMomentGroup; i += kWarps) {
    const int64_t begin = first + static_cast<int64_t>(i) * kMomentGroup, at = begin + lane * kLane;
    if (begin >= t.size) break;  // alike in a warp
    const bool whole = aligned && at + kLane <= t.size;
    Group<kHalf, kEight> group;
    group.load(t, grad, at, lane, whole);
    group.update(h);
    group.store(t, at, lane, whole, h.step_word);
  }
}

__global__ void __launch_bounds__(kThreads) adamw_kinds_kernel(const AdamWTensor* __restrict__ tensors, const uint64_t* __restrict__ grads,
                                                               const int2* __restrict__ chunks, int num_chunks, const AdamWStep h) {
  for (int c = blockIdx.x; c < num_chunks; c += gridDim.x) {
    const int2 place = chunks[c];
    const AdamWTensor t = tensors[place.x];
    const void* grad = reinterpret_cast<const void*>(grads[place.x]);
    if (t.eight) {
      if (t.half) chunk_of<true, true>(t, grad, h, place.y);
      else chunk_of<false, true>(t, grad, h, place.y);
    } else {
      if (t.half) chunk_of<true, false>(t, grad, h, place.y);
      else chunk_of<false, false>(t, grad, h, place.y);
    }
  }
}

}  // namespace

cudaError_t launch_adamw_kinds(const AdamWTensor* tensors, const uint64_t* grads, const int2* chunks, int num_chunks, const AdamWStep& h, cudaStream_t s,
                               int max_ctas) {
  if (num_chunks <= 0) return cudaSuccess;
  note_launch();
  adamw_kinds_kernel<<<max_ctas > 0 && max_ctas < num_chunks ? max_ctas : num_chunks, kThreads, 0, s>>>(tensors, grads, chunks, num_chunks, h);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace mccl
