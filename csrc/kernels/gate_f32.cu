// What stands between the fp32 products of a gated feed-forward block (sm_100a): h = act(g) u, and dg = dh u act'(g),
// du = dh act(g), in one pass each.  act(z) = z s(z), see gate.cuh.
// Bound by memory: 12 and 20 bytes a number.
#include <algorithm>

#include "kernels/gate.cuh"
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kSms = 148;

// Rows of g and of u, `ld` numbers apart, `cols` of each; h and dh have theirs one behind the other.
struct Rows {
  const float *g, *u;
  int64_t ld, rows, cols;
  bool vec, silu;
};
__global__ void __launch_bounds__(kThreads) gate_forward_kernel(const Rows w, float* __restrict__ h) {
  auto one = [&](float z, float y) { return z * gate_of(z, w.silu) * y; };
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 4;
  if (col >= w.cols) return;
  for (int64_t row = blockIdx.y; row < w.rows; row += gridDim.y) {
    const float *g = w.g + row * w.ld + col, *u = w.u + row * w.ld + col;
    float* to = h + row * w.cols + col;
    if (w.vec) {
      const float4 a = *reinterpret_cast<const float4*>(g), b = *reinterpret_cast<const float4*>(u);
      *reinterpret_cast<float4*>(to) = make_float4(one(a.x, b.x), one(a.y, b.y), one(a.z, b.z), one(a.w, b.w));
    } else {
      for (int i = 0; i < 4 && col + i < w.cols; ++i) to[i] = one(g[i], u[i]);
    }
  }
}

__global__ void __launch_bounds__(kThreads) gate_backward_kernel(const Rows w, const float* __restrict__ dh, float* __restrict__ dgu) {
  auto one = [&](float z, float y, float d, float& a, float& b) {
    const float s = gate_of(z, w.silu), t = s * (1.f - s);
    b = d * (z * s);
    // (where the curve is flat the cubic's slope may be infinite)
    a = d * y * (t > 0.f ? s + z * t * (w.silu ? 1.f : kGelu * (1.f + 3.f * kCubic * z * z)) : s);
  };
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * 4;
  if (col >= w.cols) return;
  for (int64_t row = blockIdx.y; row < w.rows; row += gridDim.y) {
    const float *g = w.g + row * w.ld + col, *u = w.u + row * w.ld + col, *d = dh + row * w.cols + col;
    float *dg = dgu + row * 2 * w.cols + col, *du = dg + w.cols;
    if (w.vec) {
      const float4 z = *reinterpret_cast<const float4*>(g), y = *reinterpret_cast<const float4*>(u), x = *reinterpret_cast<const float4*>(d);
      float4 a, b;
      one(z.x, y.x, x.x, a.x, b.x);
      one(z.y, y.y, x.y, a.y, b.y);
      one(z.z, y.z, x.z, a.z, b.z);
      one(z.w, y.w, x.w, a.w, b.w);
      *reinterpret_cast<float4*>(dg) = a;
      *reinterpret_cast<float4*>(du) = b;
    } else {
      for (int i = 0; i < 4 && col + i < w.cols; ++i) one(g[i], u[i], d[i], dg[i], du[i]);
    }
  }
}

dim3 grid_for(const Rows& w) {
  const int64_t across = (w.cols + 4 * kThreads - 1) / (4 * kThreads);
  return dim3(static_cast<unsigned>(across), static_cast<unsigned>(std::min<int64_t>(w.rows, std::max<int64_t>(1, 16 * kSms / across))));
}
Rows rows_of(const float* g, const float* u, int64_t ld, int64_t rows, int64_t cols, GatedActivation act, std::initializer_list<const void*> others) {
  uintptr_t all = reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(u);
  for (const void* p : others) all |= reinterpret_cast<uintptr_t>(p);
  return {g, u, ld, rows, cols, all % 16 == 0 && cols % 4 == 0 && ld % 4 == 0, act == GatedActivation::kSilu};
}

}  // namespace

cudaError_t launch_gate_f32(const float* g, const float* u, int64_t ld, float* h, int64_t rows, int64_t cols, GatedActivation act, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  const Rows w = rows_of(g, u, ld, rows, cols, act, {h});
  note_launch();
  gate_forward_kernel<<<grid_for(w), kThreads, 0, s>>>(w, h);
  return cudaGetLastError();
}
cudaError_t launch_gate_f32_backward(const float* gu, const float* dh, float* dgu, int64_t rows, int64_t cols, GatedActivation act, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  const Rows w = rows_of(gu, gu + cols, 2 * cols, rows, cols, act, {dh, dgu});
  note_launch();
  gate_backward_kernel<<<grid_for(w), kThreads, 0, s>>>(w, dh, dgu);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace mccl
