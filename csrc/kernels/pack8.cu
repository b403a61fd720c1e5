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

constexpr int kThreads = 256, kLanes = 8;       // threads of a block, and of a group: eight numbers each
constexpr int kUnits = kThreads / kLanes;       // groups a block has in hand at a time

// Where group `at` of the whole lies.
struct Place {
  int64_t row;
  int group;
};
__device__ __forceinline__ Place place_of(int64_t at, int64_t groups, bool few) {
  const int64_t row = few ? static_cast<int64_t>(static_cast<uint32_t>(at) / static_cast<uint32_t>(groups)) : at / groups;
  return {row, static_cast<int>(at - row * groups)};
}

// Bound by memory: one pass, 2 (4) bytes read and 1 + 1/16 written for each number.  Eight lanes share a group, so a warp
// reads 512 (1024) bytes in a run; kDeep groups are in flight for each of them before the first is looked at.
template <typename T, int kDeep>
__global__ void __launch_bounds__(kThreads) pack8_kernel(const T* __restrict__ x, int64_t ld, bool vec, const Packed8Rows p) {
  const int64_t groups = (p.cols + kGroup8 - 1) / kGroup8, all = p.rows * groups;
  const bool few = all <= 0xFFFFFFFFll;
  const int sub = threadIdx.x % kLanes;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kUnits * kDeep); base < all;
       base += static_cast<int64_t>(gridDim.x) * (kUnits * kDeep)) {
    const int64_t first = base + threadIdx.x / kLanes;
    float v[kDeep][8];
    Place at[kDeep];
    int n[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = first + d * kUnits;
      at[d] = place_of(u < all ? u : 0, groups, few);
      const int64_t left = p.cols - at[d].group * static_cast<int64_t>(kGroup8) - sub * 8;
      n[d] = u < all ? static_cast<int>(min(max(left, static_cast<int64_t>(0)), static_cast<int64_t>(8))) : 0;
      load_run<T, 8>(x + at[d].row * ld + at[d].group * static_cast<int64_t>(kGroup8) + sub * 8, n[d], vec, v[d]);
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = most8(most, v[d][i]);
#pragma unroll
      for (int m = kLanes / 2; m > 0; m /= 2) most = most8(most, __shfl_xor_sync(0xFFFFFFFFu, most, m));
      const Scale8 s = scale8(most);
      if (first + d * kUnits >= all) continue;
      const int64_t col = at[d].group * static_cast<int64_t>(kGroup8) + sub * 8;
      if (col < p.pitch)
        *reinterpret_cast<uint2*>(p.codes + at[d].row * p.pitch + col) =
            make_uint2(codes8(v[d][0], v[d][1], v[d][2], v[d][3], s.inverse), codes8(v[d][4], v[d][5], v[d][6], v[d][7], s.inverse));
      if (sub == 0) p.scales[at[d].row * groups + at[d].group] = s.scale;
    }
  }
}

template <typename T, int kDeep>
__global__ void __launch_bounds__(kThreads) unpack8_kernel(const Packed8Rows p, T* __restrict__ x, int64_t ld, bool vec) {
  const int64_t groups = (p.cols + kGroup8 - 1) / kGroup8, all = p.rows * groups;
  const bool few = all <= 0xFFFFFFFFll;
  const int sub = threadIdx.x % kLanes;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * (kUnits * kDeep) + threadIdx.x / kLanes; first < all;
       first += static_cast<int64_t>(gridDim.x) * (kUnits * kDeep)) {
    uint2 word[kDeep];
    float scale[kDeep];
    T* to[kDeep];
    int n[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = first + d * kUnits;
      const Place at = place_of(u < all ? u : 0, groups, few);
      const int64_t col = at.group * static_cast<int64_t>(kGroup8) + sub * 8, left = p.cols - col;
      n[d] = u < all ? static_cast<int>(min(max(left, static_cast<int64_t>(0)), static_cast<int64_t>(8))) : 0;
      word[d] = n[d] > 0 ? __ldcs(reinterpret_cast<const uint2*>(p.codes + at.row * p.pitch + col)) : make_uint2(0u, 0u);
      scale[d] = n[d] > 0 ? p.scales[at.row * groups + at.group] : 0.f;
      to[d] = x + at.row * ld + col;
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = value8(i < 4 ? word[d].x : word[d].y, i & 3, scale[d]);
      store_run<T, 8>(to[d], n[d], vec, v);
    }
  }
}

constexpr int kSms = 148;
int blocks_for(const Packed8Rows& p, int deep) {
  const int64_t all = p.rows * pack8_groups(p.cols), per = static_cast<int64_t>(kUnits) * deep;
  return static_cast<int>(std::min<int64_t>((all + per - 1) / per, 8 * kSms));
}
bool wide(const void* p, int64_t ld, size_t size) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * static_cast<int64_t>(size) % 16 == 0;
}

template <typename T>
cudaError_t pack(const void* x, int64_t ld, const Packed8Rows& p, cudaStream_t s) {
  constexpr int kDeep = 4;
  note_launch();
  pack8_kernel<T, kDeep><<<blocks_for(p, kDeep), kThreads, 0, s>>>(static_cast<const T*>(x), ld, wide(x, ld, sizeof(T)), p);
  return cudaGetLastError();
}
template <typename T>
cudaError_t unpack(const Packed8Rows& p, void* x, int64_t ld, cudaStream_t s) {
  constexpr int kDeep = 4;
  note_launch();
  unpack8_kernel<T, kDeep><<<blocks_for(p, kDeep), kThreads, 0, s>>>(p, static_cast<T*>(x), ld, wide(x, ld, sizeof(T)));
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
