// What the products of few rows share (gated_few.cu, linear_few.cu): matrix instructions fed as the rows lie, and runs of rows of any alignment.
#pragma once

#include <cstdint>
#include <type_traits>

#include "kernels/elems.cuh"

namespace mccl {
namespace kern {
namespace {

template <typename T>
__device__ __forceinline__ void multiply(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 numbers of a row from a column that is a multiple of 8; zeros beyond the row.  Rows that are aligned to 16 bytes are whole runs,
// and no branch stands between one load and the next.
enum class Rows { kWhole, kPadded, kAny };
template <Rows kRows, typename T>
struct Run {
  uint4 v;
  __device__ __forceinline__ void load(const T* row, int64_t at, int64_t depth, bool there, const T*, const T*) {
    const bool in = there && at < depth;
    v = *reinterpret_cast<const uint4*>(row + (in ? at : 0));
    if (!in) v = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ uint4 get(const T*) const { return v; }
};
// Aligned rows that can be read beyond their end, where there are no numbers.
template <typename T>
struct Run<Rows::kPadded, T> {
  uint4 v;
  __device__ __forceinline__ void load(const T* row, int64_t at, int64_t depth, bool there, const T*, const T*) {
    const bool in = there && at < depth;
    v = *reinterpret_cast<const uint4*>(row + (in ? at : 0));
    const int64_t n = in ? depth - at : 0;
    v.x &= n > 1 ? 0xFFFFFFFFu : n > 0 ? 0xFFFFu : 0u;
    v.y &= n > 3 ? 0xFFFFFFFFu : n > 2 ? 0xFFFFu : 0u;
    v.z &= n > 5 ? 0xFFFFFFFFu : n > 4 ? 0xFFFFu : 0u;
    v.w &= n > 7 ? 0xFFFFFFFFu : n > 6 ? 0xFFFFu : 0u;
  }
  __device__ __forceinline__ uint4 get(const T*) const { return v; }
};
// Of other rows the two aligned runs that hold the 8, moved into place when they are used; one by one where these are not inside of
// the matrix, `begin` to `end`, or the row ends.
template <typename T>
struct Run<Rows::kAny, T> {
  uint4 v, behind;
  bool moved;
  __device__ __forceinline__ void load(const T* row, int64_t at, int64_t depth, bool there, const T* begin, const T* end) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row + at);
    const uint16_t* base = p - reinterpret_cast<uintptr_t>(p) % 16 / 2;
    moved = there && at + 8 <= depth && base >= reinterpret_cast<const uint16_t*>(begin) && base + 16 <= reinterpret_cast<const uint16_t*>(end);
    if (moved) {
      v = reinterpret_cast<const uint4*>(base)[0];
      behind = reinterpret_cast<const uint4*>(base)[1];
    } else {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (there && at + i < depth) w[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i % 2));
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ uint4 get(const T* row) const {  // the row, for where it begins
    const uint32_t m = moved ? reinterpret_cast<uintptr_t>(row) % 16 : 0;
    uint32_t w[8] = {v.x, v.y, v.z, v.w, behind.x, behind.y, behind.z, behind.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = m & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = m & 4 ? w[i + 1] : w[i];
    const uint32_t bits = m & 2 ? 16 : 0;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                      __funnelshift_r(w[3], w[4], bits));
  }
};

}  // namespace
}  // namespace kern
}  // namespace mccl
