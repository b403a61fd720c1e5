// Activation checkpoints in 8 bits (sm_100a).
//
// Of each group of 64 numbers of a row: s = max|x| / 127, code = rint(x (127 / max|x|)), and back code s.  A group with an
// infinity or a NaN comes back as NaN, one without a number of 2^-100 as zeros.
#include <algorithm>

#include "kernels/elems.cuh"
#include "kernels/launch_count.h"
#include "kernels/pack8_api.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kLanes = 4;       // threads of a block, and of a group: two runs of eight numbers each, 32 apart
constexpr int kUnits = kThreads / kLanes;       // groups a block has in hand at a time
constexpr int kDeep = 2;                        // groups of a thread in flight
constexpr int kTurn = kUnits * kDeep;           // groups of a block's turn

// Where a group lies.  Rows that are whole groups, one behind the other, are one row.
struct Steps {
  int64_t all, groups;    // of the whole, of a row
};
struct Place {
  int64_t row;
  int64_t col;
  __device__ __forceinline__ Place(const Steps& t, int64_t unit, bool linear) {
    if (linear) {
      row = 0;
      col = unit * kGroup8;
    } else {
      row = t.all <= 0xFFFFFFFFll ? static_cast<uint32_t>(unit) / static_cast<uint32_t>(t.groups) : unit / t.groups;
      col = (unit - row * t.groups) * kGroup8;
    }
  }
};
__device__ __forceinline__ int present(int64_t cols, int64_t col, bool there) {
  return there ? static_cast<int>(min(max(cols - col, static_cast<int64_t>(0)), static_cast<int64_t>(8))) : 0;
}

// Bound by memory: one pass, 2 (4) bytes read and 1 + 1/16 written for each number.  Four lanes share a group, so that few
// instructions are spent on what a group needs once; kDeep groups of each are in flight before the first is looked at.
template <typename T, bool kLinear>
__global__ void __launch_bounds__(kThreads, 4) pack8_kernel(const T* __restrict__ x, int64_t ld, bool vec, const Packed8Rows p, const Steps t) {
  const int sub = threadIdx.x % kLanes;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTurn; base < t.all; base += static_cast<int64_t>(gridDim.x) * kTurn) {
    const int64_t unit = base + threadIdx.x / kLanes;
    float v[kDeep][2][8];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
      const Place at(t, u < t.all ? u : 0, kLinear);
      const int64_t col = at.col + sub * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const T* from = x + at.row * ld + col + 32 * h;
        load_run<T, 8>(from, kLinear ? (u < t.all ? 8 : 0) : present(p.cols, col + 32 * h, u < t.all), kLinear || vec, v[d][h]);
      }
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      uint32_t bits = 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = most8(bits, v[d][h][i]);
#pragma unroll
      for (int m = kLanes / 2; m > 0; m /= 2) bits = max(bits, __shfl_xor_sync(0xFFFFFFFFu, bits, m));
      // scale8, its two quotients in two lanes
      const float most = __uint_as_float(bits);
      const bool finite = most < INFINITY, kept = finite && most >= kTiny8;
      const float quotient = __fdiv_rn(sub == 0 ? most : 127.f, sub == 0 ? 127.f : most);
      const float shared = __shfl_sync(0xFFFFFFFFu, quotient, 1, kLanes), inverse = kept ? shared : 0.f;
      const int64_t u = unit + d * kUnits;
      if (u >= t.all) continue;
      const Place at(t, u, kLinear);
      const int64_t col = at.col + sub * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (kLinear || col + 32 * h < p.pitch)
          *reinterpret_cast<uint2*>(p.codes + at.row * p.pitch + col + 32 * h) =
              make_uint2(codes8(v[d][h][0], v[d][h][1], v[d][h][2], v[d][h][3], inverse), codes8(v[d][h][4], v[d][h][5], v[d][h][6], v[d][h][7], inverse));
      if (sub == 0) p.scales[u] = kept ? quotient : finite ? 0.f : NAN;
    }
  }
}

template <typename T, bool kLinear>
__global__ void __launch_bounds__(kThreads, 4) unpack8_kernel(const Packed8Rows p, T* __restrict__ x, int64_t ld, bool vec, const Steps t) {
  const int sub = threadIdx.x % kLanes;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kTurn + threadIdx.x / kLanes; unit < t.all; unit += static_cast<int64_t>(gridDim.x) * kTurn) {
    uint2 word[kDeep][2];
    float scale[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
      const bool there = u < t.all;
      const Place at(t, there ? u : 0, kLinear);
      const int64_t col = at.col + sub * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        word[d][h] = there && (kLinear || col + 32 * h < p.cols) ? __ldcs(reinterpret_cast<const uint2*>(p.codes + at.row * p.pitch + col + 32 * h))
                                                                 : make_uint2(0u, 0u);
      scale[d] = there ? p.scales[u] : 0.f;
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
      const Place at(t, u < t.all ? u : 0, kLinear);
      const int64_t col = at.col + sub * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = value8(i < 4 ? word[d][h].x : word[d][h].y, i & 3, scale[d]);
        store_run<T, 8>(x + at.row * ld + col + 32 * h, kLinear ? (u < t.all ? 8 : 0) : present(p.cols, col + 32 * h, u < t.all), kLinear || vec, v);
      }
    }
  }
}

constexpr int kSms = 148;
struct Shape {
  int blocks;
  bool vec, linear;
  Steps t;
};
// One row (`linear`) where rows are whole groups that follow each other, aligned: no division, no ends inside of a group.
Shape shape_of(const Packed8Rows& p, const void* x, int64_t ld, size_t size) {
  Shape s{};
  s.vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * static_cast<int64_t>(size) % 16 == 0;
  s.linear = s.vec && p.cols % kGroup8 == 0 && p.pitch == p.cols && (ld == p.cols || p.rows == 1);
  s.t.groups = pack8_groups(p.cols);
  s.t.all = p.rows * s.t.groups;
  s.blocks = static_cast<int>(std::min<int64_t>((s.t.all + kTurn - 1) / kTurn, 32 * kSms));
  return s;
}

template <typename T>
cudaError_t pack(const void* x, int64_t ld, const Packed8Rows& p, cudaStream_t s) {
  const Shape h = shape_of(p, x, ld, sizeof(T));
  note_launch();
  if (h.linear) pack8_kernel<T, true><<<h.blocks, kThreads, 0, s>>>(static_cast<const T*>(x), ld, h.vec, p, h.t);
  else pack8_kernel<T, false><<<h.blocks, kThreads, 0, s>>>(static_cast<const T*>(x), ld, h.vec, p, h.t);
  return cudaGetLastError();
}
template <typename T>
cudaError_t unpack(const Packed8Rows& p, void* x, int64_t ld, cudaStream_t s) {
  const Shape h = shape_of(p, x, ld, sizeof(T));
  note_launch();
  if (h.linear) unpack8_kernel<T, true><<<h.blocks, kThreads, 0, s>>>(p, static_cast<T*>(x), ld, h.vec, h.t);
  else unpack8_kernel<T, false><<<h.blocks, kThreads, 0, s>>>(p, static_cast<T*>(x), ld, h.vec, h.t);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_pack8(const void* x, Elem type, int64_t ld, const Packed8Rows& p, cudaStream_t s) {
  if (p.rows <= 0 || p.cols <= 0) return cudaSuccess;
  if (p.pitch < p.cols || p.pitch % 16 != 0 || (reinterpret_cast<uintptr_t>(p.codes) & 7) != 0) return cudaErrorInvalidValue;
  switch (type) {
    case Elem::kF32: return pack<float>(x, ld, p, s);
    case Elem::kF16: return pack<__half>(x, ld, p, s);
    default: return pack<__nv_bfloat16>(x, ld, p, s);
  }
}
cudaError_t launch_unpack8(const Packed8Rows& p, void* x, Elem type, int64_t ld, cudaStream_t s) {
  if (p.rows <= 0 || p.cols <= 0) return cudaSuccess;
  if (p.pitch < p.cols || p.pitch % 16 != 0 || (reinterpret_cast<uintptr_t>(p.codes) & 7) != 0) return cudaErrorInvalidValue;
  switch (type) {
    case Elem::kF32: return unpack<float>(p, x, ld, s);
    case Elem::kF16: return unpack<__half>(p, x, ld, s);
    default: return unpack<__nv_bfloat16>(p, x, ld, s);
  }
}

}  // namespace kern
}  // namespace mccl
