// Linear layer for few rows, such as one token of each of a few sequences, with bias, activation and residual (sm_100a).
//
// Bound by the weights' way from memory.  A block has 8 or 16 rows of the weights, its warps share the reduction; a lane reads 8 numbers of a
// weight row and 8 of a token's and gives them to the matrix instructions as they are: which of the 32 numbers of a step is called k = 0 does not
// matter as long as both operands agree.  With 8 rows half of an instruction's rows are zeros, which it costs nothing: it is the loads that count.
//
// us from memory, bf16 (B200): 1 token of 1024 x 1024 2.5, 1024 x 4096 6.1, 4096 x 4096 11.4 (2.9 TB/s), 16384 x 1024 18; 16 tokens of 2048 x 2048 5.5; rows
// that begin anywhere, 1723 x 5258, 16 (both sides of where tiles are faster beside layer_is_few).
#include "kernels/elems.cuh"
#include "kernels/few.cuh"
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"
#include "kernels/layer_act.cuh"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kStep = 32, kSms = 148;  // k of a step of one warp

struct Few {
  const void *x, *w;
  int64_t ldx, ldw, in, out;
  int tokens;
  LayerFinish f;
  void* y;
};

// kGroups groups of 8 tokens (the last ones may be none); kRows 8 or 16 rows of weights.
template <typename T, int kGroups, int kRows, bool kVec>
__global__ void __launch_bounds__(kThreads, kGroups == 4 ? 1 : 2) layer_few_kernel(const Few w) {
  constexpr int kW = kRows / 8, kAhead = kVec ? (kW == 1 && kGroups == 1 ? 8 : 4) : 2, kHeld = 2 * kW;
  __shared__ float part[kWarps][kGroups][kHeld][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const T *x = static_cast<const T*>(w.x), *weights = static_cast<const T*>(w.w);
  const T* weight[kW];  // of rows that there are not, the first one
  bool there[kW];
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    there[i] = first + 8 * i + g < w.out;
    weight[i] = weights + (there[i] ? first + 8 * i + g : 0) * w.ldw;
  }
  const T* token[kGroups];  // of tokens that there are not, the first one's
#pragma unroll
  for (int n = 0; n < kGroups; ++n) token[n] = x + (8 * n + g < w.tokens ? 8 * n + g : 0) * w.ldx;
  const int64_t begin = warp * kStep + t * 8, step = kWarps * kStep;
  float sum[kGroups][4];
#pragma unroll
  for (int n = 0; n < kGroups; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
  for (int64_t at = begin; at < w.in + t * 8; at += kAhead * step) {  // alike in a warp's lanes
    Run<kVec ? Rows::kWhole : Rows::kAny, T> run[kAhead][kW];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int i = 0; i < kW; ++i) run[a][i].load(weight[i], at + a * step, w.in, there[i], weights, weights + (w.out - 1) * w.ldw + w.in);
    uint4 rows[kAhead][kW];  // moved once for all tokens
    if constexpr (!kVec)
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
#pragma unroll
        for (int i = 0; i < kW; ++i) rows[a][i] = run[a][i].get(weight[i]);
#pragma unroll
    for (int n = 0; n < kGroups; ++n) {
      Run<kVec ? Rows::kWhole : Rows::kAny, T> b[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) b[a].load(token[n], at + a * step, w.in, true, x, x + (w.tokens - 1) * w.ldx + w.in);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const uint4 a0 = kVec ? run[a][0].v : rows[a][0], y = b[a].get(token[n]);
        const uint4 a1 = kW == 1 ? make_uint4(0u, 0u, 0u, 0u) : kVec ? run[a][kW - 1].v : rows[a][kW - 1];
        multiply<T>(sum[n], a0.x, a1.x, a0.y, a1.y, y.x, y.y);
        multiply<T>(sum[n], a0.z, a1.z, a0.w, a1.w, y.z, y.w);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kGroups; ++n)
#pragma unroll
    for (int i = 0; i < kHeld; ++i) part[warp][n][i][lane] = sum[n][i];
  __syncthreads();
  // a lane has rows g and 8 + g, tokens 2 t and 2 t + 1 of a group; neighbouring threads have neighbouring rows of y
  for (int item = threadIdx.x; item < kGroups * 8 * kRows; item += kThreads) {
    const int r = item % kRows, m = item / kRows, n = m / 8, i = r / 8 * 2 + m % 2, at = r % 8 * 4 + m % 8 / 2;
    const int64_t row = first + r;
    float z = 0.f;
#pragma unroll
    for (int p = 0; p < kWarps; ++p) z += part[p][n][i][at];
    if (m >= w.tokens || row >= w.out) continue;
    if (w.f.bias != nullptr) z += Traits<T>::load(static_cast<const T*>(w.f.bias)[row]);
    const float a = with_activation(w.f.activation, [&](auto act) { return Act16::value<decltype(act)::kValue>(z); });
    const int64_t to = m * w.out + row, from = m * w.f.ldr + row;
    if (w.f.y_f32) static_cast<float*>(w.y)[to] = w.f.residual == nullptr ? a : a + static_cast<const float*>(w.f.residual)[from];
    else static_cast<T*>(w.y)[to] = Traits<T>::store(w.f.residual == nullptr ? a : a + Traits<T>::load(static_cast<const T*>(w.f.residual)[from]));
  }
}

template <typename T, int kRows, bool kVec>
void run(const Few& w, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((w.out + kRows - 1) / kRows);
  if (w.tokens <= 8) layer_few_kernel<T, 1, kRows, kVec><<<blocks, kThreads, 0, s>>>(w);
  else if (w.tokens <= 16) layer_few_kernel<T, 2, kRows, kVec><<<blocks, kThreads, 0, s>>>(w);
  else layer_few_kernel<T, 4, kRows, kVec><<<blocks, kThreads, 0, s>>>(w);
}
template <typename T>
cudaError_t launch(const LayerFew& g, cudaStream_t s) {
  const Few w{g.x.data, g.weight.data, g.x.ld, g.weight.ld, g.in, g.out, static_cast<int>(g.tokens), g.finish, g.y};
  auto aligned = [](const GatedOperand& m, int64_t rows) { return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && (rows <= 1 || m.ld % 8 == 0); };
  const bool vec = g.in % 8 == 0 && aligned(g.x, g.tokens) && aligned(g.weight, g.out), more = g.out >= 16 * 4 * kSms;
  note_launch();
  if (vec) more ? run<T, 16, true>(w, s) : run<T, 8, true>(w, s);
  else more ? run<T, 16, false>(w, s) : run<T, 8, false>(w, s);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_layer_few(const LayerFew& g, cudaStream_t s) {
  if (g.tokens <= 0 || g.tokens > kFewTokens || g.in <= 0 || g.out <= 0 || g.in > 0x7FFFFFFFll || g.out > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  return g.bf16 ? launch<__nv_bfloat16>(g, s) : launch<__half>(g, s);
}

}  // namespace kern
}  // namespace mccl
