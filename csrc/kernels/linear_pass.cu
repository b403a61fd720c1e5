// What stands around the products of a linear layer (sm_100a): activation and residual behind an fp32 product, and before the products of the
// backward pass dz = dy act'(z) with its sums over the rows, the gradient of the bias, in the same pass and before dz is rounded.
// Bound by memory: each number is read and written once.  dz and the bias's gradient of 8192 x 4096 bf16 behind gelu 35 us (201 MB: 5.8 TB/s) and 3 for
// the blocks' sums; the sums alone of 8192 x 1024 fp32 13.
#include <algorithm>
#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"
#include "kernels/layer_act.cuh"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kSms = 148;
constexpr int kRowsAhead = 4;     // of a warp, in flight
constexpr int kJoinThreads = 1024;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- fp32: y = act(z) + residual ------------------------------------------------------------------------------
struct Finish {
  const float *z, *residual;
  int64_t ldr, rows, cols;
  float* y;
};
template <LayerActivation kAct, int kV>
__global__ void __launch_bounds__(kThreads) layer_finish_kernel(const Finish w) {
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kV;
  if (col >= w.cols) return;
  for (int64_t row = blockIdx.y; row < w.rows; row += gridDim.y) {
    float v[kV], r[kV];
    load_run<float, kV>(w.z + row * w.cols + col, kV, true, v);
    if (w.residual != nullptr) load_run<float, kV>(w.residual + row * w.ldr + col, kV, true, r);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      v[i] = Act32::value<kAct>(v[i]);
      if (w.residual != nullptr) v[i] += r[i];
    }
    store_run<float, kV>(w.y + row * w.cols + col, kV, true, v);
  }
}

// ---- dz and the bias's gradient ---------------------------------------------------------------------------------
// kV numbers of a row, as they lie in memory.
template <typename T, int kV>
struct RawRun {
  static constexpr int kBytes = kV * sizeof(T);
  using Word = std::conditional_t<kBytes >= 16, uint4, std::conditional_t<kBytes == 8, uint2, T>>;
  Word w[kBytes >= 16 ? kBytes / 16 : 1];
  __device__ __forceinline__ void load(const T* p) {
    const Word* f = reinterpret_cast<const Word*>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / sizeof(Word)); ++i) w[i] = f[i];
  }
  __device__ __forceinline__ float operator[](int i) const { return Traits<T>::load(reinterpret_cast<const T*>(w)[i]); }
};
// T: the operands' type; D: of dy.  A warp has kV columns a lane, and every kWarps-th row of its block's; kRowsAhead of them are asked for while the
// ones before are worked on.
template <typename T, typename D, LayerActivation kAct, int kV>
__global__ void __launch_bounds__(kThreads, 2) layer_derive_kernel(const LayerDerive g, int64_t rows_each) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  using Act = std::conditional_t<std::is_same_v<T, float>, Act32, Act16>;
  constexpr bool kSlope = kAct != LayerActivation::kNone;
  __shared__ float sums[kWarps][32 * kV];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * kV, begin = blockIdx.y * rows_each, end = min(g.rows, begin + rows_each);
  float sum[kV];
#pragma unroll
  for (int i = 0; i < kV; ++i) sum[i] = 0.f;
  if (col < g.cols) {
    const D* dy = static_cast<const D*>(g.dy.data) + col;
    const T* z = static_cast<const T*>(g.z.data) + col;
    T* dz = static_cast<T*>(g.dz) + col;
    RawRun<D, kV> next_d[kRowsAhead];
    RawRun<T, kV> next_z[kRowsAhead];
    auto ask = [&](int r, int64_t at) {
      if (at >= end) return;
      next_d[r].load(dy + at * g.dy.ld);
      if constexpr (kSlope) next_z[r].load(z + at * g.z.ld);
    };
#pragma unroll
    for (int r = 0; r < kRowsAhead; ++r) ask(r, begin + warp + r * kWarps);
#pragma unroll 1
    for (int64_t row = begin + warp; row < end; row += kRowsAhead * kWarps) {
#pragma unroll
      for (int r = 0; r < kRowsAhead; ++r) {  // each place is asked for again as soon as its numbers are in registers of their own
        const int64_t at = row + r * kWarps;
        if (at >= end) break;
        float d[kV], v[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          d[i] = next_d[r][i];
          if constexpr (kSlope) v[i] = next_z[r][i];
        }
        ask(r, at + kRowsAhead * kWarps);
        if constexpr (kV > 1 && !std::is_same_v<T, float>) {
#pragma unroll
          for (int i = 0; i < kV; i += 2) {
            if constexpr (kSlope) derived<Act, kAct>(Two(d[i], d[i + 1]), Two(v[i], v[i + 1])).apart(d[i], d[i + 1]);
            add_to<2>(sum + i, d + i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            if constexpr (kSlope) d[i] = derived<Act, kAct>(d[i], v[i]);
            sum[i] += d[i];
          }
        }
        if (g.dz != nullptr) store_run<T, kV>(dz + at * g.dz_ld, kV, true, d);
      }
    }
  }
  if (g.bias == nullptr) return;
#pragma unroll
  for (int i = 0; i < kV; ++i) sums[warp][lane * kV + i] = sum[i];
  __syncthreads();
  float* to = g.partial + blockIdx.y * g.cols;
  for (int i = threadIdx.x; i < 32 * kV; i += kThreads) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 * kV + i;
    if (c >= g.cols) continue;
    float all = 0.f;
#pragma unroll
    for (int p = 0; p < kWarps; ++p) all += sums[p][i];
    if (gridDim.y == 1) static_cast<T*>(g.bias)[c] = Traits<T>::store(all);  // of few rows the one block's are the whole sums
    else to[c] = all;
  }
}
// Adds up the blocks' sums: 32 columns a block, whose warps share the parts.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) layer_join_kernel(const float* partial, int parts, int64_t cols, T* bias) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kParts = kJoinThreads / 32;
  __shared__ float sums[kParts][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float sum = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int p = warp; p < parts; p += kParts) sum += __ldcg(partial + p * cols + c);
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp > 0 || c >= cols) return;
  for (int i = 1; i < kParts; ++i) sum += sums[i][lane];
  bias[c] = Traits<T>::store(sum);
}

int64_t parts_of(int64_t rows, int64_t cols) { return std::clamp<int64_t>(ceil_div(4 * kSms, ceil_div(cols, 256)), 1, std::max<int64_t>(1, ceil_div(rows, 4 * kWarps))); }

template <typename T, typename D, int kV>
cudaError_t derive(const LayerDerive& g, cudaStream_t s) {
  const int64_t parts = parts_of(g.rows, g.cols);
  const dim3 grid(static_cast<unsigned>(ceil_div(g.cols, 32 * kV)), static_cast<unsigned>(parts));
  note_launch();
  with_activation(g.activation, [&](auto act) { layer_derive_kernel<T, D, decltype(act)::kValue, kV><<<grid, kThreads, 0, s>>>(g, ceil_div(g.rows, parts)); });
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || g.bias == nullptr || parts == 1) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(g.cols, 32)));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, layer_join_kernel<T>, static_cast<const float*>(g.partial), static_cast<int>(parts), g.cols, static_cast<T*>(g.bias));
}
template <typename T, typename D>
cudaError_t derive(const LayerDerive& g, cudaStream_t s) {
  constexpr int kV = 16 / sizeof(D);  // 8 numbers of 16 bits, 4 beside numbers of 32
  auto aligned = [](const void* p, int64_t ld, int size) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (kV * size) == 0 && ld % kV == 0); };
  if (g.cols % kV == 0 && aligned(g.dy.data, g.dy.ld, sizeof(D)) && aligned(g.z.data, g.z.ld, sizeof(T)) && aligned(g.dz, g.dz_ld, sizeof(T))) return derive<T, D, kV>(g, s);
  return derive<T, D, 1>(g, s);
}
template <typename T>
cudaError_t derive(const LayerDerive& g, cudaStream_t s) {
  return g.dy.type == Elem::kF32 ? derive<T, float>(g, s) : derive<T, T>(g, s);
}

}  // namespace

cudaError_t launch_layer_finish(const float* z, const LayerRows& residual, float* y, int64_t rows, int64_t cols, LayerActivation act, cudaStream_t s) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  const Finish w{z, static_cast<const float*>(residual.data), residual.ld, rows, cols, y};
  const uintptr_t all = reinterpret_cast<uintptr_t>(z) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(residual.data);
  const bool vec = all % 16 == 0 && cols % 4 == 0 && (residual.data == nullptr || residual.ld % 4 == 0);
  const int64_t across = ceil_div(cols, (vec ? 4 : 1) * kThreads);
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(std::min<int64_t>(rows, std::max<int64_t>(1, 16 * kSms / across))));
  note_launch();
  with_activation(act, [&](auto a) {
    if (vec) layer_finish_kernel<decltype(a)::kValue, 4><<<grid, kThreads, 0, s>>>(w);
    else layer_finish_kernel<decltype(a)::kValue, 1><<<grid, kThreads, 0, s>>>(w);
  });
  return cudaGetLastError();
}

int64_t layer_partial_bytes(int64_t rows, int64_t cols) { return 4 * parts_of(rows, cols) * cols; }

cudaError_t launch_layer_derive(const LayerDerive& g, cudaStream_t s) {
  if (g.rows <= 0 || g.cols <= 0) return cudaSuccess;
  if ((g.activation == LayerActivation::kNone) != (g.z.data == nullptr)) return cudaErrorInvalidValue;
  if (g.z.data != nullptr && g.z.type != g.dz_type) return cudaErrorInvalidValue;
  if (g.dy.type != Elem::kF32 && g.dy.type != g.dz_type) return cudaErrorInvalidValue;
  if (g.bias != nullptr && g.bias_type != g.dz_type) return cudaErrorInvalidValue;
  return g.dz_type == Elem::kF32 ? derive<float, float>(g, s) : g.dz_type == Elem::kBF16 ? derive<__nv_bfloat16>(g, s) : derive<__half>(g, s);
}

}  // namespace kern
}  // namespace mccl
