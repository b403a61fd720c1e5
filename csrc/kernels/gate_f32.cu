// What stands between the fp32 products of a gated feed-forward block (sm_100a): h = act(g) u, and dg = dh u act'(g),
// du = dh act(g), in one pass each.  act(z) = z s(z), see gated.cu; here with exponential and quotient to the last bits.
// Bound by memory: 12 and 20 bytes a number.
#include <algorithm>

#include "kernels/gated_api.h"
#include "kernels/launch_count.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kSms = 148;
constexpr float kGelu = 1.5957691216057308f, kCubic = 0.044715f;  // 2 sqrt(2 / pi)

__device__ __forceinline__ float gate_of(float z, bool silu) { return 1.f / (1.f + expf(-(silu ? z : kGelu * (z + kCubic * z * z * z)))); }

__global__ void __launch_bounds__(kThreads) gate_forward_kernel(const float* __restrict__ g, const float* __restrict__ u, float* __restrict__ h,
                                                                int64_t n, bool vec, bool silu) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kThreads;
  auto one = [&](float z, float y) { return z * gate_of(z, silu) * y; };
  const int64_t runs = vec ? n / 4 : 0;
  for (int64_t i = at; i < runs; i += step) {
    const float4 a = reinterpret_cast<const float4*>(g)[i], b = reinterpret_cast<const float4*>(u)[i];
    reinterpret_cast<float4*>(h)[i] = make_float4(one(a.x, b.x), one(a.y, b.y), one(a.z, b.z), one(a.w, b.w));
  }
  for (int64_t i = 4 * runs + at; i < n; i += step) h[i] = one(g[i], u[i]);
}

__global__ void __launch_bounds__(kThreads) gate_backward_kernel(const float* __restrict__ g, const float* __restrict__ u, const float* __restrict__ dh,
                                                                 float* __restrict__ dg, float* __restrict__ du, int64_t n, bool vec, bool silu) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kThreads;
  auto one = [&](float z, float y, float d, float& a, float& b) {
    const float s = gate_of(z, silu), t = s * (1.f - s);
    b = d * (z * s);
    // (where the curve is flat the cubic's slope may be infinite)
    a = d * y * (t > 0.f ? s + z * t * (silu ? 1.f : kGelu * (1.f + 3.f * kCubic * z * z)) : s);
  };
  const int64_t runs = vec ? n / 4 : 0;
  for (int64_t i = at; i < runs; i += step) {
    const float4 z = reinterpret_cast<const float4*>(g)[i], y = reinterpret_cast<const float4*>(u)[i], d = reinterpret_cast<const float4*>(dh)[i];
    float4 a, b;
    one(z.x, y.x, d.x, a.x, b.x);
    one(z.y, y.y, d.y, a.y, b.y);
    one(z.z, y.z, d.z, a.z, b.z);
    one(z.w, y.w, d.w, a.w, b.w);
    reinterpret_cast<float4*>(dg)[i] = a;
    reinterpret_cast<float4*>(du)[i] = b;
  }
  for (int64_t i = 4 * runs + at; i < n; i += step) one(g[i], u[i], dh[i], dg[i], du[i]);
}

int blocks_for(int64_t n) { return static_cast<int>(std::min<int64_t>((n + 4 * kThreads - 1) / (4 * kThreads), 8 * kSms)); }
bool wide(std::initializer_list<const void*> ps) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= reinterpret_cast<uintptr_t>(p);
  return all % 16 == 0;
}

}  // namespace

cudaError_t launch_gate_f32(const float* g, const float* u, float* h, int64_t n, GatedActivation act, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  note_launch();
  gate_forward_kernel<<<blocks_for(n), kThreads, 0, s>>>(g, u, h, n, wide({g, u, h}), act == GatedActivation::kSilu);
  return cudaGetLastError();
}
cudaError_t launch_gate_f32_backward(const float* g, const float* u, const float* dh, float* dg, float* du, int64_t n, GatedActivation act,
                                     cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  note_launch();
  gate_backward_kernel<<<blocks_for(n), kThreads, 0, s>>>(g, u, dh, dg, du, n, wide({g, u, dh, dg, du}), act == GatedActivation::kSilu);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace mccl
