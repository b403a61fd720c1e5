// What both passes of layer norm (norm_forward.cu, norm_backward.cu) share: a team's row in registers, its types, sums over the team.
#pragma once

#include <algorithm>
#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/launch_count.h"
#include "kernels/norm_api.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kSms = 148;
constexpr int kFew = 8, kMany = 16;                           // numbers of a row that a thread has
constexpr int kForwardThreads = 512, kBackwardThreads = 512;  // of a block, at most
constexpr int kWideThreads = 512;
constexpr int kForwardBlocks = 2 * kSms, kBackwardBlocks = 2 * kSms;  // that stay

// An array's type: known where the kernel is compiled, or one that it is told.  The usual sets of types have kernels of their own: with types that
// are looked up a number took 50 instructions of the forward pass, 28 us of 8192 x 1024 for 17.
template <Elem kType>
struct Is {
  __device__ __forceinline__ explicit Is(Elem) {}
  __device__ __forceinline__ constexpr operator Elem() const { return kType; }
};
struct Told {
  Elem type;
  __device__ __forceinline__ explicit Told(Elem t) : type(t) {}
  __device__ __forceinline__ operator Elem() const { return type; }
};
template <typename X, typename S, typename Y, typename W>
struct Types {
  static constexpr int kRun = 4;  // numbers of a run where rows are aligned: 16 bytes of the widest
};
using F = Is<Elem::kF32>;
using H = Is<Elem::kF16>;
using B = Is<Elem::kBF16>;
template <>
struct Types<B, B, B, F> { static constexpr int kRun = 8; };
template <>
struct Types<H, H, H, F> { static constexpr int kRun = 8; };
template <>
struct Types<B, B, B, B> { static constexpr int kRun = 8; };
template <>
struct Types<H, H, H, H> { static constexpr int kRun = 8; };
using AnyTypes = Types<Told, Told, Told, Told>;
// Calls `f` with the types of x, of the stream, of y and of the weights.
template <typename Call>
cudaError_t with_types(Elem x, Elem s, Elem y, Elem w, Call f) {
  auto are = [&](Elem a, Elem b, Elem c, Elem d) { return x == a && s == b && y == c && w == d; };
  constexpr Elem kF = Elem::kF32, kH = Elem::kF16, kB = Elem::kBF16;
  if (are(kF, kF, kF, kF)) return f(Types<F, F, F, F>());
  if (are(kF, kF, kB, kF)) return f(Types<F, F, B, F>());
  if (are(kF, kF, kH, kF)) return f(Types<F, F, H, F>());
  if (are(kB, kF, kB, kF)) return f(Types<B, F, B, F>());
  if (are(kH, kF, kH, kF)) return f(Types<H, F, H, F>());
  if (are(kB, kB, kB, kF)) return f(Types<B, B, B, F>());
  if (are(kH, kH, kH, kF)) return f(Types<H, H, H, F>());
  if (are(kB, kB, kB, kB)) return f(Types<B, B, B, B>());
  if (are(kH, kH, kH, kH)) return f(Types<H, H, H, H>());
  return f(AnyTypes());
}

// kRun numbers that are aligned to their run's size (16 bytes at most).
template <int kRun>
__device__ __forceinline__ void put(void* p, Elem type, int64_t at, const float (&v)[kRun]) {
  if (type == Elem::kF32) store_run<float, kRun>(static_cast<float*>(p) + at, kRun, true, v);
  else if (type == Elem::kBF16) store_run<__nv_bfloat16, kRun>(static_cast<__nv_bfloat16*>(p) + at, kRun, true, v);
  else store_run<__half, kRun>(static_cast<__half*>(p) + at, kRun, true, v);
}
// A thread's runs of a row, every `team`th, so that neighbours have neighbouring runs: as they come from memory, and as numbers.  What is
// loaded is not looked at before all of it is asked for: with the conversion behind each load, in the branch that knows the type, every
// array's way from memory was waited for by itself.
template <int kRun, int kN>
struct Raw {
  uint32_t w[kN][kRun];  // of 16 bits two a word, or with runs of one one
  template <typename T>
  __device__ __forceinline__ void load(const void* p, T type, int64_t at, int t, int team, int cols) {
    if (type == Elem::kF32) {
      const uint32_t* f = static_cast<const uint32_t*>(p) + at;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int c = (n * team + t) * kRun;
        if constexpr (kRun == 1) {
          w[n][0] = c < cols ? f[c] : 0u;
        } else {
#pragma unroll
          for (int i = 0; i < kRun; i += 4) {
            const uint4 x = c < cols ? *reinterpret_cast<const uint4*>(f + c + i) : make_uint4(0u, 0u, 0u, 0u);
            w[n][i] = x.x, w[n][i + 1] = x.y, w[n][i + 2] = x.z, w[n][i + 3] = x.w;
          }
        }
      }
    } else {
      const uint16_t* f = static_cast<const uint16_t*>(p) + at;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int c = (n * team + t) * kRun;
        if constexpr (kRun == 1) {
          w[n][0] = c < cols ? f[c] : 0u;
        } else if constexpr (kRun == 4) {
          const uint2 x = c < cols ? *reinterpret_cast<const uint2*>(f + c) : make_uint2(0u, 0u);
          w[n][0] = x.x, w[n][1] = x.y;
        } else {
          const uint4 x = c < cols ? *reinterpret_cast<const uint4*>(f + c) : make_uint4(0u, 0u, 0u, 0u);
          w[n][0] = x.x, w[n][1] = x.y, w[n][2] = x.z, w[n][3] = x.w;
        }
      }
    }
  }
};
template <int kRun, int kN>
struct Row {
  float v[kN][kRun];
  template <typename T>
  __device__ __forceinline__ void take(const Raw<kRun, kN>& raw, T type) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        const uint32_t word = type == Elem::kF32 || kRun == 1 ? raw.w[n][i] : raw.w[n][i / 2];
        const uint32_t half = i % 2 ? word >> 16 : word & 0xFFFFu;
        v[n][i] = type == Elem::kF32 ? __uint_as_float(word) : type == Elem::kBF16 ? __uint_as_float(half << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(half)));
      }
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) v[n][i] = x;
  }
  template <typename T>
  __device__ __forceinline__ void put(T* p, int t, int team, int cols) const {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int c = (n * team + t) * kRun;
      if (c < cols) store_run<T, kRun>(p + c, kRun, true, v[n]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(void* p, T type, int64_t at, int t, int team, int cols) const {
    if (type == Elem::kF32) put(static_cast<float*>(p) + at, t, team, cols);
    else if (type == Elem::kBF16) put(static_cast<__nv_bfloat16*>(p) + at, t, team, cols);
    else put(static_cast<__half*>(p) + at, t, team, cols);
  }
  // As the type keeps it.
  template <typename T>
  __device__ __forceinline__ void round(T type) {
    if (type != Elem::kF32)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          v[n][i] = type == Elem::kBF16 ? __bfloat162float(__float2bfloat16_rn(v[n][i])) : __half2float(__float2half_rn(v[n][i]));
  }
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
  return x;
}
// Sums over a team of warps, the same bits in all of its threads.  Two slots in turn: a warp writes one again only behind the barrier that all
// others reach behind reading it.
struct Team {
  float2* slots;  // [2][warps of the block]
  int warps, first, number, turn;
  __device__ __forceinline__ Team(float2* s, int warps_of, int block_warps) : slots(s), warps(warps_of), turn(0) {
    number = threadIdx.x / 32 / warps;
    first = number * warps;
    all = block_warps;
  }
  int all;
  __device__ __forceinline__ float2 sum(float a, float b) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (warps == 1) return make_float2(a, b);
    float2* mine = slots + turn * all + first;
    turn ^= 1;
    if (threadIdx.x % 32 == 0) mine[threadIdx.x / 32 - first] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(number + 1), "r"(32 * warps) : "memory");
    float2 r = mine[0];
    for (int i = 1; i < warps; ++i) {
      const float2 x = mine[i];
      r.x += x.x;
      r.y += x.y;
    }
    return r;
  }
  __device__ __forceinline__ float sum(float a) {
    if (warps == 1) return warp_sum(a);
    return sum(a, 0.f).x;
  }
};

// ---- host ---------------------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int size_of(Elem e) { return e == Elem::kF32 ? 4 : 2; }

// The longest run that all arrays are aligned to: 8 numbers, 4 or one.
struct Alignment {
  int run;
  explicit Alignment(int cols) : run(cols % 8 == 0 ? 8 : cols % 4 == 0 ? 4 : 1) {}
  void with(const void* p, int64_t ld, Elem type) {
    if (p == nullptr) return;
    while (run > 1 && (reinterpret_cast<uintptr_t>(p) % std::min(16, run * size_of(type)) != 0 || ld % run != 0)) run = run == 8 ? 4 : 1;
  }
};
// Calls `f` with the types and the run of a kernel for them: that of the types, one, or, between the two, four of any types.
template <typename T, typename Call>
cudaError_t with_run(T types, int run, Call f) {
  if (run >= T::kRun) return f(types, std::integral_constant<int, T::kRun>());
  if (run == 1) return f(types, std::integral_constant<int, 1>());
  return f(AnyTypes(), std::integral_constant<int, 4>());
}

int block_warps(int warps, int most) { return warps * std::max(1, most / warps); }

// Rows that are read one number at a time have kernels for teams of so many warps and numbers a thread, known where they are compiled: places are then a
// distance from one address, and a thread asks for no more numbers than a row of its kind has.  (8192 x 1024 and the like, by runs, are faster
// with the team that just holds them, and the addresses are few.)  Calls `f` with the warps and the numbers of the smallest team.
template <typename Call>
cudaError_t with_team(int cols, Call f) {
  auto is = [&](auto warps, auto numbers) { return f(warps, numbers); };
#define TEAM(w, n) \
  if (cols <= 32 * w * n) return is(std::integral_constant<int, w>(), std::integral_constant<int, n>())
  TEAM(1, 1);
  TEAM(1, 2);
  TEAM(1, 4);
  TEAM(1, 8);
  TEAM(2, 8);
  TEAM(4, 8);
  TEAM(8, 6);
  TEAM(8, 8);
  TEAM(16, 8);
  TEAM(16, 12);
  TEAM(16, 16);
#undef TEAM
  return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace kern
}  // namespace mccl
