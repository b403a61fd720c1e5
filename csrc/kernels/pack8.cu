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

constexpr int kThreads = 256;

// ---- rows that are whole groups, one behind the other, aligned: one long row --------------------------------------
constexpr int kLanes = 4;                       // threads of a group: two runs of eight numbers each, 32 apart
constexpr int kUnits = kThreads / kLanes;       // groups a block has in hand at a time
constexpr int kDeep = 2;                        // groups of a thread in flight
constexpr int kTurn = kUnits * kDeep;           // groups of a block's turn

// A group's scale, in the lane `sub` 0 of it, and what its numbers are multiplied with, from the bits of its largest magnitude: scale8
// with its two quotients in two lanes.
struct Shared8 {
  float scale, inverse;
};
template <int kOver>
__device__ __forceinline__ Shared8 shared8(uint32_t bits, int sub) {
#pragma unroll
  for (int m = kOver / 2; m > 0; m /= 2) bits = max(bits, __shfl_xor_sync(0xFFFFFFFFu, bits, m));
  const float most = __uint_as_float(bits);
  const bool finite = most < INFINITY, kept = finite && most >= kTiny8;
  const float quotient = __fdiv_rn(sub == 0 ? most : 127.f, sub == 0 ? 127.f : most);
  const float inverse = __shfl_sync(0xFFFFFFFFu, quotient, 1, kOver);
  return {kept ? quotient : finite ? 0.f : NAN, kept ? inverse : 0.f};
}

// Bound by memory: one pass, 2 (4) bytes read and 1 + 1/16 written for each number.  Four lanes share a group, so that few
// instructions are spent on what a group needs once; kDeep groups of each are in flight before the first is looked at.
// 16384 x 5632 bf16 to codes 46 us, back 40 (B200; 5.9 and 6.7 TB/s).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) pack8_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scales, int64_t all) {
  const int sub = threadIdx.x % kLanes;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTurn; base < all; base += static_cast<int64_t>(gridDim.x) * kTurn) {
    const int64_t unit = base + threadIdx.x / kLanes;
    float v[kDeep][2][8];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
#pragma unroll
      for (int h = 0; h < 2; ++h) load_run<T, 8>(x + u * kGroup8 + sub * 8 + 32 * h, u < all ? 8 : 0, true, v[d][h]);
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      uint32_t bits = 0u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = most8(bits, v[d][h][i]);
      const Shared8 s = shared8<kLanes>(bits, sub);
      const int64_t u = unit + d * kUnits;
      if (u >= all) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<uint2*>(codes + u * kGroup8 + sub * 8 + 32 * h) =
            make_uint2(codes8(v[d][h][0], v[d][h][1], v[d][h][2], v[d][h][3], s.inverse), codes8(v[d][h][4], v[d][h][5], v[d][h][6], v[d][h][7], s.inverse));
      if (sub == 0) scales[u] = s.scale;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) unpack8_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ x, int64_t all) {
  const int sub = threadIdx.x % kLanes;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kTurn + threadIdx.x / kLanes; unit < all; unit += static_cast<int64_t>(gridDim.x) * kTurn) {
    uint2 word[kDeep][2];
    float scale[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
#pragma unroll
      for (int h = 0; h < 2; ++h) word[d][h] = u < all ? __ldcs(reinterpret_cast<const uint2*>(codes + u * kGroup8 + sub * 8 + 32 * h)) : make_uint2(0u, 0u);
      scale[d] = u < all ? scales[u] : 0.f;
    }
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const int64_t u = unit + d * kUnits;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        values8(word[d][h].x, scale[d], v);
        values8(word[d][h].y, scale[d], v + 4);
        store_run<T, 8>(x + u * kGroup8 + sub * 8 + 32 * h, u < all ? 8 : 0, true, v);
      }
    }
  }
}

// ---- any rows -----------------------------------------------------------------------------------------------------
// Sixteen lanes share a group and have every sixteenth of its numbers, so that neighbours read and write neighbours wherever a row
// begins.  (Runs of eight a lane, one number at a time: 9349 x 2731 fp16 to codes and back 141 us.)
constexpr int kWideLanes = 16, kEach = kGroup8 / kWideLanes, kWideUnits = kThreads / kWideLanes, kWideDeep = 4;

// Where a group lies.  Steps from one to the next are divided by the groups of a row on the host.
struct Place {
  int64_t row;
  int group;
};
struct Steps {
  int64_t all, groups;    // of the whole, of a row
  int64_t unit_rows, turn_rows;
  int unit_groups, turn_groups;   // from one of a thread's groups to the next, and from one of its turns
};
__device__ __forceinline__ Place onward(const Place& p, int64_t rows, int by, const Steps& t) {
  Place n{p.row + rows, p.group + by};
  if (n.group >= t.groups) {
    n.group -= static_cast<int>(t.groups);
    ++n.row;
  }
  return n;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack8_rows_kernel(const T* __restrict__ x, int64_t ld, const Packed8Rows p, const Steps t) {
  const int sub = threadIdx.x % kWideLanes;
  constexpr int kStep = kWideUnits * kWideDeep;
  int64_t unit = static_cast<int64_t>(blockIdx.x) * kStep + threadIdx.x / kWideLanes;
  Place turn{unit / t.groups, 0};
  turn.group = static_cast<int>(unit - turn.row * t.groups);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kStep; base < t.all;
       base += static_cast<int64_t>(gridDim.x) * kStep, unit += static_cast<int64_t>(gridDim.x) * kStep) {
    float v[kWideDeep][kEach];
    Place at = turn;
#pragma unroll
    for (int d = 0; d < kWideDeep; ++d) {
      const int64_t col = at.group * static_cast<int64_t>(kGroup8) + sub;
      const T* from = x + at.row * ld + col;
      const int64_t left = unit + d * kWideUnits < t.all ? p.cols - col : 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) v[d][i] = kWideLanes * i < left ? Traits<T>::load(from[kWideLanes * i]) : 0.f;
      at = onward(at, t.unit_rows, t.unit_groups, t);
    }
    at = turn;
#pragma unroll
    for (int d = 0; d < kWideDeep; ++d) {
      uint32_t bits = 0u;
#pragma unroll
      for (int i = 0; i < kEach; ++i) bits = most8(bits, v[d][i]);
      const Shared8 s = shared8<kWideLanes>(bits, sub);
      const uint32_t word = codes8(v[d][0], v[d][1], v[d][2], v[d][3], s.inverse);
      if (unit + d * kWideUnits < t.all) {
        const int64_t col = at.group * static_cast<int64_t>(kGroup8) + sub;
        int8_t* to = p.codes + at.row * p.pitch + col;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (col + kWideLanes * i < p.pitch) to[kWideLanes * i] = static_cast<int8_t>(word >> (8 * i));
        if (sub == 0) p.scales[at.row * t.groups + at.group] = s.scale;
      }
      at = onward(at, t.unit_rows, t.unit_groups, t);
    }
    turn = onward(turn, t.turn_rows, t.turn_groups, t);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack8_rows_kernel(const Packed8Rows p, T* __restrict__ x, int64_t ld, const Steps t) {
  const int sub = threadIdx.x % kWideLanes;
  constexpr int kStep = kWideUnits * kWideDeep;
  int64_t unit = static_cast<int64_t>(blockIdx.x) * kStep + threadIdx.x / kWideLanes;
  Place turn{unit / t.groups, 0};
  turn.group = static_cast<int>(unit - turn.row * t.groups);
  for (; unit < t.all; unit += static_cast<int64_t>(gridDim.x) * kStep) {
    int8_t code[kWideDeep][kEach];
    float scale[kWideDeep];
    Place at = turn;
#pragma unroll
    for (int d = 0; d < kWideDeep; ++d) {
      const int64_t col = at.group * static_cast<int64_t>(kGroup8) + sub, left = unit + d * kWideUnits < t.all ? p.cols - col : 0;
      const int8_t* from = p.codes + at.row * p.pitch + col;
#pragma unroll
      for (int i = 0; i < kEach; ++i) code[d][i] = kWideLanes * i < left ? from[kWideLanes * i] : static_cast<int8_t>(0);
      scale[d] = left > 0 ? p.scales[at.row * t.groups + at.group] : 0.f;
      at = onward(at, t.unit_rows, t.unit_groups, t);
    }
    at = turn;
#pragma unroll
    for (int d = 0; d < kWideDeep; ++d) {
      const int64_t col = at.group * static_cast<int64_t>(kGroup8) + sub, left = unit + d * kWideUnits < t.all ? p.cols - col : 0;
      T* to = x + at.row * ld + col;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (kWideLanes * i < left) to[kWideLanes * i] = Traits<T>::store(static_cast<float>(code[d][i]) * scale[d]);
      at = onward(at, t.unit_rows, t.unit_groups, t);
    }
    turn = onward(turn, t.turn_rows, t.turn_groups, t);
  }
}

constexpr int kSms = 148;
int blocks_for(int64_t all, int per) { return static_cast<int>(std::min<int64_t>((all + per - 1) / per, 32 * kSms)); }
// Rows that are whole groups, follow each other and are aligned.
bool one_row(const Packed8Rows& p, const void* x, int64_t ld, size_t size) {
  return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && p.cols % kGroup8 == 0 && p.pitch == p.cols && (ld == p.cols || p.rows == 1) &&
         p.cols * static_cast<int64_t>(size) % 16 == 0;
}
Steps steps_of(const Packed8Rows& p, int& blocks) {
  Steps t{};
  constexpr int kStep = kWideUnits * kWideDeep;
  t.groups = pack8_groups(p.cols);
  t.all = p.rows * t.groups;
  blocks = blocks_for(t.all, kStep);
  t.unit_rows = kWideUnits / t.groups;
  t.unit_groups = static_cast<int>(kWideUnits % t.groups);
  t.turn_rows = static_cast<int64_t>(blocks) * kStep / t.groups;
  t.turn_groups = static_cast<int>(static_cast<int64_t>(blocks) * kStep % t.groups);
  return t;
}

template <typename T>
cudaError_t pack(const void* x, int64_t ld, const Packed8Rows& p, cudaStream_t s) {
  note_launch();
  if (one_row(p, x, ld, sizeof(T))) {
    const int64_t all = p.rows * pack8_groups(p.cols);
    pack8_kernel<T><<<blocks_for(all, kTurn), kThreads, 0, s>>>(static_cast<const T*>(x), p.codes, p.scales, all);
  } else {
    int blocks = 0;
    const Steps t = steps_of(p, blocks);
    pack8_rows_kernel<T><<<blocks, kThreads, 0, s>>>(static_cast<const T*>(x), ld, p, t);
  }
  return cudaGetLastError();
}
template <typename T>
cudaError_t unpack(const Packed8Rows& p, void* x, int64_t ld, cudaStream_t s) {
  note_launch();
  if (one_row(p, x, ld, sizeof(T))) {
    const int64_t all = p.rows * pack8_groups(p.cols);
    unpack8_kernel<T><<<blocks_for(all, kTurn), kThreads, 0, s>>>(p.codes, p.scales, static_cast<T*>(x), all);
  } else {
    int blocks = 0;
    const Steps t = steps_of(p, blocks);
    unpack8_rows_kernel<T><<<blocks, kThreads, 0, s>>>(p, static_cast<T*>(x), ld, t);
  }
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
