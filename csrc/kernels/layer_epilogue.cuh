// What follows a linear layer's product in the kernels that have it in tensor memory (gated.cu, linear_tiles.cu): bias, activation and residual of
// a warp's 32 rows, 64 columns at a time, and the boxes in shared memory that z and y leave from.
#pragma once

#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/layer_act.cuh"
#include "kernels/tensor_pipe.cuh"

namespace mccl {
namespace kern {
namespace {

struct Layer {
  LayerActivation activation;
  const char *bias, *residual;
  int64_t ldr, cols;
  bool bias_vec, residual_vec;  // aligned to 16 bytes, whole runs of them
};
bool residual_aligned(const LayerFinish& f, int64_t cols) {
  const int64_t size = f.y_f32 ? 4 : 2;
  return cols * size % 16 == 0 && f.ldr * size % 16 == 0 && f.ldr >= cols && reinterpret_cast<uintptr_t>(f.residual) % 16 == 0;
}

Layer layer_of(const LayerFinish& f, int64_t cols) {
  return {f.activation, static_cast<const char*>(f.bias), static_cast<const char*>(f.residual), f.ldr, cols,
          cols % 8 == 0 && reinterpret_cast<uintptr_t>(f.bias) % 16 == 0, residual_aligned(f, cols)};
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kBf16) return store_pair<__nv_bfloat16>(a, b);
  else return store_pair<__half>(a, b);
}

constexpr int kTurn = 64, kBoxBytes = 32 * kTurn * 2;
template <bool kBf16>
struct Staged {
  uint32_t row;       // of the first box
  int swizzle;
  __device__ __forceinline__ Staged(uint32_t boxes, int lane) : row(boxes + lane * 128), swizzle(lane & 7) {}
  __device__ __forceinline__ void put(int which, int i, const float* v) const {
    const uint32_t to = row + which * kBoxBytes + ((i / 8) ^ swizzle) * 16;
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pack2<kBf16>(v[0], v[1])), "r"(pack2<kBf16>(v[2], v[3])),
                 "r"(pack2<kBf16>(v[4], v[5])), "r"(pack2<kBf16>(v[6], v[7]))
                 : "memory");
  }
  __device__ __forceinline__ uint4 get(int which, int i) const {  // 8 numbers as they were put
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(row + which * kBoxBytes + ((i / 8) ^ swizzle) * 16)
                 : "memory");
    return v;
  }
  // In 32 bits: boxes of 32 columns, from the `which`th on.
  __device__ __forceinline__ void put_f32(int which, int i, const float* v) const {
    const uint32_t box = row + (which + i / 32) * kBoxBytes;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(box + ((((i % 32) + e) / 4) ^ swizzle) * 16), "f"(v[e]), "f"(v[e + 1]), "f"(v[e + 2]),
                   "f"(v[e + 3])
                   : "memory");
  }
  __device__ __forceinline__ void get_f32(int which, int i, float* v) const {  // as they were put
    const uint32_t box = row + (which + i / 32) * kBoxBytes;
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[e]), "=f"(v[e + 1]), "=f"(v[e + 2]), "=f"(v[e + 3])
                   : "r"(box + ((((i % 32) + e) / 4) ^ swizzle) * 16)
                   : "memory");
  }
};
// 16 bytes from `from` on, numbers of kSize bytes of which there are `n`.
template <int kSize>
__device__ __forceinline__ uint4 run_of(const char* from, int64_t n, bool vec) {
  constexpr int kPer = 16 / kSize;
  if (vec) return n > 0 ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0u, 0u, 0u, 0u);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < n) {
      if constexpr (kSize == 4) w[i] = reinterpret_cast<const uint32_t*>(from)[i];
      else w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(from)[i]) << (16 * (i % 2));
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A warp's residual of a turn, 32 rows of 64 columns, by whole runs of the rows, where a thread's own row would take 32 requests for each of its runs.
// Its place in y's boxes is where y's numbers go.  In 16 bits it waits in registers until the boxes are free; in 32, where sums have the
// registers, aligned rows come by themselves (load_own_box), others through here.
struct LayerResidual {
  static constexpr int kWords = 32, kLanes = kTurn * 2 / 16, kRowsAt = 32 / kLanes;  // lanes of a row, and rows a request, of aligned ones
  uint32_t w[kWords];
  // Rows from `row` on of `rows`, columns from `col` on.
  __device__ __forceinline__ void load(const Layer& l, int64_t row, int64_t rows, int64_t col, int lane) {
    const char* from = l.residual + 2 * (row * l.ldr + col);
    const int64_t n = l.cols - col;
    const int high = static_cast<int>(min(rows - row, static_cast<int64_t>(32)));
    if (l.residual_vec) {
      const int at = lane % kLanes * 8, left = at < n ? high - lane / kLanes : 0;
      const char* to = from + 2 * (lane / kLanes * l.ldr + at);
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i, to += 2 * kRowsAt * l.ldr) {
        const uint4 v = i * kRowsAt < left ? __ldcs(reinterpret_cast<const uint4*>(to)) : make_uint4(0u, 0u, 0u, 0u);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else {
      const char* to = from + 4 * lane;  // two neighbours
      const bool one = 2 * lane < n, two = 2 * lane + 1 < n;
#pragma unroll
      for (int r = 0; r < 32; ++r, to += 2 * l.ldr) {
        const uint32_t a = r < high && one ? reinterpret_cast<const uint16_t*>(to)[0] : 0u, b = r < high && two ? reinterpret_cast<const uint16_t*>(to)[1] : 0u;
        w[r] = a | b << 16;
      }
    }
  }
  __device__ __forceinline__ void put(bool vec, int lane, uint32_t box) const {
    if (vec) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const int r = i * kRowsAt + lane / kLanes;
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + r * 128 + ((lane % kLanes) ^ (r & 7)) * 16), "r"(w[4 * i]), "r"(w[4 * i + 1]),
                     "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                     : "memory");
      }
    } else {
#pragma unroll
      for (int r = 0; r < 32; ++r) asm volatile("st.shared.b32 [%0], %1;" ::"r"(box + r * 128 + ((lane / 4) ^ (r & 7)) * 16 + lane % 4 * 4), "r"(w[r]) : "memory");
    }
  }
};
// In 32 bits, rows that are not aligned: two neighbours a lane, eight rows at a time.
__device__ __forceinline__ void put_residual(const Layer& l, int64_t row, int64_t rows, int64_t col, int lane, uint32_t box) {
  const char* to = l.residual + 4 * (row * l.ldr + col + 2 * lane);
  const int64_t n = l.cols - col - 2 * lane;
  const int high = static_cast<int>(min(rows - row, static_cast<int64_t>(32)));
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 8) {
    uint32_t v[16];
#pragma unroll
    for (int r = 0; r < 8; ++r, to += 4 * l.ldr) {
      v[2 * r] = r0 + r < high && n > 0 ? reinterpret_cast<const uint32_t*>(to)[0] : 0u;
      v[2 * r + 1] = r0 + r < high && n > 1 ? reinterpret_cast<const uint32_t*>(to)[1] : 0u;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(box + lane / 16 * kBoxBytes + (r0 + r) * 128 + ((lane % 16 / 2) ^ r) * 16 + lane % 2 * 8), "r"(v[2 * r]),
                   "r"(v[2 * r + 1])
                   : "memory");
  }
  __syncwarp();
}
template <bool kBf16>
__device__ __forceinline__ void halves(const uint4& raw, float* v) {  // 8 numbers of 16 bits
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = kBf16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)) : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// 8 columns of z as they are kept: beyond fp16's range slopes are what they are at its end.
template <bool kBf16, typename Sink>
__device__ __forceinline__ void put_z(const Sink& sink, int i, const float* z) {
  if constexpr (kBf16) {
    sink.put(0, i, z);
  } else {
    float kept[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) kept[e] = z[e] != z[e] ? z[e] : fminf(fmaxf(z[e], -65504.f), 65504.f);
    sink.put(0, i, kept);
  }
}

// Where y and z go: maps of them, and y's memory for rows that are not aligned, which have no map.
struct LayerTarget {
  const CUtensorMap *y_map, *z_map;
  void* to;
  int64_t ldo, rows;
  bool wide;
};
// The boxes of 64 columns, of which there are `left`, from `col` on, of the warp's rows from `y` on, to z and y.
template <bool kKeep, bool kWide>
__device__ __forceinline__ void flush_layer(const LayerTarget& j, int64_t col, int left, int64_t y, uint32_t boxes, int lane) {
  constexpr int kFirst = kKeep ? 1 : 0;  // y's boxes behind z's
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    if (y < j.rows) {
      const int x = static_cast<int>(col);
      if constexpr (kKeep) store_box(j.z_map, boxes, x, static_cast<int>(y));
      if (j.wide) {
        store_box(j.y_map, boxes + kFirst * kBoxBytes, x, static_cast<int>(y));
        if (kWide && left > 32) store_box(j.y_map, boxes + (kFirst + 1) * kBoxBytes, x + 32, static_cast<int>(y));
      }
    }
    stores_commit();
  }
  if (!j.wide) {  // rows that are not aligned: two numbers a lane, row by row
    const int n = static_cast<int>(min(static_cast<int64_t>(32), j.rows - y)), here = left - 2 * lane;
    char* to = static_cast<char*>(j.to) + (y * j.ldo + col + 2 * lane) * (kWide ? 4 : 2);
#pragma unroll 4
    for (int r = 0; r < n; ++r, to += j.ldo * (kWide ? 4 : 2)) {
      uint32_t v[2];
      if constexpr (kWide) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1])
                     : "r"(boxes + (kFirst + lane / 16) * kBoxBytes + r * 128 + ((lane % 16 / 2) ^ (r & 7)) * 16 + lane % 2 * 8));
        if (here > 0) reinterpret_cast<uint32_t*>(to)[0] = v[0];
        if (here > 1) reinterpret_cast<uint32_t*>(to)[1] = v[1];
      } else {
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[0]) : "r"(boxes + kFirst * kBoxBytes + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4));
        if (here > 0) reinterpret_cast<uint16_t*>(to)[0] = static_cast<uint16_t>(v[0]);
        if (here > 1) reinterpret_cast<uint16_t*>(to)[1] = static_cast<uint16_t>(v[0] >> 16);
      }
    }
    __syncwarp();
  }
}

}  // namespace
}  // namespace kern
}  // namespace mccl
