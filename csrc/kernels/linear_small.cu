// Linear layer of small fp32 matrices, forward with bias, activation and residual, backward with both products and the bias's gradient: one launch each
// (sm_100a), where products of their own, one behind the other, are mostly their launches.
//
// c(i, j) = sum over k of a(i, k) b(j, k) in fp32, by multiplications and additions.  Bound by the launch and by the way along k, about 1.1 us for each 64.
// A block has 32 x 32 of c; its four groups of 64 threads share each 64 of k, a thread has 4 x 4, and the next 64 are on their way meanwhile.  The
// groups' sums are added in a fixed order.
//
// us on the device, and the library's products and sums in brackets (B200): forward 136 x 128 x 128 5.2 (6.3), 656 x 77 x 176 5.4 (6.2), 3 x 256 x 192 6.5 (2.7), 1024 x
// 256 x 256 11.4 (9.8), and 2 to 3 more in brackets behind an activation; backward 8.3 (13), 20 (24), 6.6 (8.2), 34 (35).  The host
// gets there in 9 us and 57 (autograd's engine included) where the library's calls and the passes around them take 15 to 19 and 90.
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"
#include "kernels/layer_act.cuh"

namespace mccl {
namespace kern {
namespace {

constexpr int kTile = 32, kDepth = 64, kThreads = 256, kPitch = kTile + 1, kEach = kTile * kDepth / kThreads;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One operand: a(i, k) at i * step_i + k * step_k, one of which is 1.
struct Operand {
  const float* data;
  int64_t step_i, step_k, rows;
};
// What a thread holds of 32 rows and 64 of k, neighbours along what is contiguous; to shared memory as [k][i].  kInner: k is.
template <bool kInner>
struct Held {
  static constexpr int kRow = kInner ? kThreads / kDepth : 0, kK = kInner ? 0 : kThreads / kTile;  // from one of its numbers to the next
  float v[kEach];
  const float* from;  // its first number's, of this stage
  int64_t apart, next, left;
  int i, k;
  uint32_t rows;  // which of its numbers are of rows that there are
  __device__ __forceinline__ Held(const Operand& m, int64_t begin, int64_t depth) {
    i = kInner ? threadIdx.x / kDepth : threadIdx.x % kTile;
    k = kInner ? threadIdx.x % kDepth : threadIdx.x / kTile;
    from = m.data + (begin + i) * m.step_i + k * m.step_k;
    apart = kInner ? kRow * m.step_i : kK * m.step_k;
    next = kDepth * m.step_k;
    left = depth - k;
    rows = 0u;
#pragma unroll
    for (int e = 0; e < kEach; ++e) rows |= begin + i + e * kRow < m.rows ? 1u << e : 0u;
  }
  // The next stage's.
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = (rows >> e & 1u) && e * kK < left ? from[e * apart] : 0.f;
    from += next;
    left -= kDepth;
  }
  __device__ __forceinline__ void put(float* to) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) to[(k + e * kK) * kPitch + i + e * kRow] = v[e];
  }
};
struct Product {
  Operand a, b;
  int64_t depth;
  int tiles_j, blocks;
  float* sums;  // of a's rows, or null
};
struct Work {
  Product job[2];
  LayerActivation activation;
  const float *bias, *residual;  // forward's
  int64_t ldr;
  float *z, *to[2];  // rows of b's rows
};

// kA, kB: k is contiguous in a and in b.  `job`: which of the backward pass's two.
template <bool kForward, bool kA, bool kB>
__device__ __forceinline__ void multiply(const Work& w, int job, int tile, float* as, float* bs) {
  const Product& p = w.job[job];
  const int64_t begin_a = static_cast<int64_t>(tile / p.tiles_j) * kTile, begin_b = static_cast<int64_t>(tile % p.tiles_j) * kTile;
  const int group = threadIdx.x / 64, ti = threadIdx.x % 8, tj = threadIdx.x % 64 / 8;
  const bool sums = !kForward && p.sums != nullptr && tile % p.tiles_j == 0;
  Held<kA> a(p.a, begin_a, p.depth);
  Held<kB> b(p.b, begin_b, p.depth);
  float c[4][4], sum = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) c[x][y] = 0.f;
  a.load();
  b.load();
  for (int64_t k0 = 0; k0 < p.depth; k0 += kDepth) {
    a.put(as);
    b.put(bs);
    __syncthreads();
    if (k0 + kDepth < p.depth) {
      a.load();
      b.load();
    }
    if (sums && threadIdx.x < kTile) {
      float part = 0.f;
#pragma unroll 8
      for (int k = 0; k < kDepth; ++k) part += as[k * kPitch + threadIdx.x];
      sum += part;
    }
#pragma unroll
    for (int k = 0; k < kDepth / 4; ++k) {
      const float *ka = as + (group * (kDepth / 4) + k) * kPitch + ti, *kb = bs + (group * (kDepth / 4) + k) * kPitch + tj;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = ka[8 * e], y[e] = kb[8 * e];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) c[e][f] = fmaf(x[e], y[f], c[e][f]);
    }
    __syncthreads();
  }
  if (sums && threadIdx.x < kTile && begin_a + threadIdx.x < p.a.rows) p.sums[begin_a + threadIdx.x] = sum;
  // the groups' parts, two behind the other two
  auto part = [&](int i, int j) -> float& { return (group & 1 ? bs : as)[i * kPitch + j]; };
#pragma unroll
  for (int turn = 1; turn >= 0; --turn) {
    if (group / 2 == turn)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          float& to = part(ti + 8 * e, tj + 8 * f);
          to = turn ? c[e][f] : to + c[e][f];
        }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < kTile * kTile / kThreads; ++e) {
    const int n = e * kThreads + threadIdx.x, r = n / kTile, col = n % kTile;
    const int64_t i = begin_a + r, j = begin_b + col;
    if (i >= p.a.rows || j >= p.b.rows) continue;
    float v = as[r * kPitch + col] + bs[r * kPitch + col];
    const int64_t to = i * p.b.rows + j;
    if constexpr (kForward) {
      if (w.bias != nullptr) v += w.bias[j];
      if (w.z != nullptr) w.z[to] = v;
      v = with_activation(w.activation, [&](auto act) { return Act32::value<decltype(act)::kValue>(v); });
      if (w.residual != nullptr) v += w.residual[i * w.ldr + j];
    }
    w.to[job][to] = v;
  }
}
template <bool kForward>
__global__ void __launch_bounds__(kThreads) layer_small_kernel(const __grid_constant__ Work w) {
  __shared__ float as[kDepth * kPitch], bs[kDepth * kPitch];
  const int block = static_cast<int>(blockIdx.x);
  if constexpr (kForward) multiply<true, true, true>(w, 0, block, as, bs);
  else if (block < w.job[0].blocks) multiply<false, true, false>(w, 0, block, as, bs);
  else multiply<false, false, false>(w, 1, block - w.job[0].blocks, as, bs);
}

void shape(Product& p) {
  p.tiles_j = static_cast<int>(ceil_div(p.b.rows, kTile));
  p.blocks = static_cast<int>(ceil_div(p.a.rows, kTile)) * p.tiles_j;
}

}  // namespace

cudaError_t launch_layer_small(const LayerSmall& g, cudaStream_t s) {
  if (g.tokens <= 0 || g.in <= 0 || g.out <= 0 || !layer_is_small(g.tokens, g.in, g.out)) return cudaErrorInvalidValue;
  Work w{};
  w.job[0] = {{g.x, g.ldx, 1, g.tokens}, {g.weight, g.ldw, 1, g.out}, g.in, 0, 0, nullptr};
  shape(w.job[0]);
  w.activation = g.activation;
  w.bias = g.bias;
  w.residual = g.residual;
  w.ldr = g.ldr;
  w.z = g.z;
  w.to[0] = g.y;
  note_launch();
  layer_small_kernel<true><<<w.job[0].blocks, kThreads, 0, s>>>(w);
  return cudaGetLastError();
}
cudaError_t launch_layer_small_backward(const LayerSmallBackward& g, cudaStream_t s) {
  if (g.tokens <= 0 || g.in <= 0 || g.out <= 0 || !layer_is_small_backward(g.tokens, g.in, g.out)) return cudaErrorInvalidValue;
  Work w{};
  const bool products[2] = {g.dx != nullptr, g.dw != nullptr || g.dbias != nullptr};
  if (products[0]) w.job[0] = {{g.dz, g.ldz, 1, g.tokens}, {g.weight, 1, g.ldw, g.in}, g.out, 0, 0, nullptr};
  if (products[1]) w.job[1] = {{g.dz, 1, g.ldz, g.out}, {g.x, 1, g.ldx, g.in}, g.tokens, 0, 0, g.dbias};
  for (int i = 0; i < 2; ++i) {
    if (products[i]) shape(w.job[i]);
    w.to[i] = i == 0 ? g.dx : g.dw;
  }
  if (g.dw == nullptr && products[1]) w.job[1].tiles_j = 1, w.job[1].b.rows = 0, w.job[1].blocks = static_cast<int>(ceil_div(g.out, kTile));  // the sums alone
  const int blocks = w.job[0].blocks + w.job[1].blocks;
  if (blocks == 0) return cudaSuccess;
  note_launch();
  layer_small_kernel<false><<<blocks, kThreads, 0, s>>>(w);
  return cudaGetLastError();
}

}  // namespace kern
}  // namespace mccl
