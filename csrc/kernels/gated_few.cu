// Gated feed-forward block for few rows, such as one token of each of a few sequences (sm_100a).
//
// Bound by the weights' way from memory, 6 bytes of them for width x hidden numbers.  A block has 8 rows of each of the two
// projections (of the projection back 8), its warps share the reduction; a lane reads 8 numbers of a weight row and 8 of a token's
// and these are what it gives to the matrix instructions: which of the 32 numbers of a step is called k = 0 does not matter as long as
// both operands agree, so nothing is rearranged.  The products are a few instructions a kilobyte; with multiplications and additions
// instead 16 tokens of 1024 x 2816 took 78 us (the tokens' numbers came from the cache for every row), and the tiles of 256 rows of
// gated.cu take 19 for any number of tokens up to 64.  h is the sum of two 16-bit numbers here, which
// leave 2^-16 of it (bf16) or 2^-22 (fp16, in its normal range).
// us (B200, weights of six blocks in turn), 1, 8, 16, 32 tokens: 1024 x 2816 8.3, 9.4, 13.4, 18.3; 2048 x 5632 18.2 (69 MB: 3.8 TB/s),
// 20.6, 31.6, 40.0; 4096 x 10240 56 (4.5 TB/s), 63, 100, 122; 1000 x 2731, whose rows of w_down begin anywhere, 10.2, 10.9, 13.7, 20.9
// (read in pairs from the first aligned number on 12.9, 17.3, 33, 42), 1723 x 5258, all rows, 37, 39, 48, 66 (47, 57, 86, 122).
// A run of a block's rows ahead of the products, 4 or 16 warps a block, more of the row in flight: all slower; so are weights through a
// ring in shared memory, 24 runs a thread on their way at any time (64 us of 4096 x 10240 and 8 tokens: what is left of the first-level
// cache doesn't hold the tokens).  16 rows a block of the projection back: 59 of it, but 24 for 21 of 2048 x 5632.
#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/gate.cuh"
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kRows = 8, kStep = 32;  // k of a step of one warp

struct Few {
  const void* x[2];    // tokens; h as its upper and lower part
  const void* w[2];
  void* out[2];
  int64_t ldx, ldw[2], ldo;
  int64_t rows, depth; // of the weights
  int tokens;
  float c0, c1;        // the curve, see gated.cu; fp32 asks for gate.cuh's
  bool silu;
};

__device__ __forceinline__ float gate(float z, float c0, float c1) {
  return 1.f / (1.f + exp2f(z * fmaf(c1, fminf(z * z, 1e30f), c0)));
}
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

// kGroups groups of 8 tokens (the last ones may be none).  kUp: gate and up and what follows them, else one product of h.
template <typename T, int kGroups, bool kUp, bool kVec>
__global__ void __launch_bounds__(kThreads, kGroups == 2 && kVec ? 3 : 2) few_kernel(const Few w) {
  constexpr int kX = kUp ? 1 : 2, kW = kUp ? 2 : 1, kAhead = !kVec ? (kUp || kGroups > 2 ? 2 : 5 - kGroups) : !kUp && kGroups == 1 ? 8 : 4;
  constexpr int kHeld = kUp ? 4 : 2;  // accumulators of a lane and group that mean something
  __shared__ float part[kWarps][kGroups][kHeld][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kRows;
  const bool there = first + g < w.rows;
  const T* weight[kW];
#pragma unroll
  for (int i = 0; i < kW; ++i) weight[i] = static_cast<const T*>(w.w[i]) + (there ? first + g : 0) * w.ldw[i];
  const int64_t begin = warp * kStep + t * 8, step = kWarps * kStep;
  Run<kVec ? Rows::kWhole : Rows::kAny, T> run[kAhead][kW];
  auto load = [&](int64_t at) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int i = 0; i < kW; ++i)
        run[a][i].load(weight[i], at + a * step, w.depth, there, static_cast<const T*>(w.w[i]), static_cast<const T*>(w.w[i]) + (w.rows - 1) * w.ldw[i] + w.depth);
  };
  // The second launch is let in behind the first one's wait: whatever wrote the weights is done by then, and their first runs are
  // asked for before h is there.
  if constexpr (!kUp) load(begin);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if constexpr (kUp) load(begin);
  float sum[kGroups][4];
#pragma unroll
  for (int n = 0; n < kGroups; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
  const T* token[kGroups][kX];  // of tokens that there are not, the first one's
#pragma unroll
  for (int n = 0; n < kGroups; ++n)
#pragma unroll
    for (int p = 0; p < kX; ++p) token[n][p] = static_cast<const T*>(w.x[p]) + (8 * n + g < w.tokens ? 8 * n + g : 0) * w.ldx;
  for (int64_t at = begin; at < w.depth + t * 8; at += kAhead * step) {  // alike in a warp's lanes
    if (at != begin) load(at);
    uint4 rows[kAhead][kW];  // moved once for all tokens
    if constexpr (!kVec)
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
#pragma unroll
        for (int i = 0; i < kW; ++i) rows[a][i] = run[a][i].get(weight[i]);
#pragma unroll
    for (int n = 0; n < kGroups; ++n) {
      Run<kVec ? Rows::kWhole : kUp ? Rows::kAny : Rows::kPadded, T> b[kAhead][kX];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
#pragma unroll
        for (int p = 0; p < kX; ++p)
          b[a][p].load(token[n][p], at + a * step, w.depth, true, static_cast<const T*>(w.x[p]), static_cast<const T*>(w.x[p]) + (w.tokens - 1) * w.ldx + w.depth);
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
#pragma unroll
        for (int p = 0; p < kX; ++p) {
          const uint4 a0 = kVec ? run[a][0].v : rows[a][0], y = b[a][p].get(token[n][p]);
          const uint4 a1 = !kUp ? make_uint4(0u, 0u, 0u, 0u) : kVec ? run[a][kW - 1].v : rows[a][kW - 1];
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
  // a lane has rows g (and of the second projection g again), tokens 2 t and 2 t + 1 of a group
  for (int item = threadIdx.x; item < kGroups * 64; item += kThreads) {
    const int at = item % 32, i = item / 32 % 2, n = item / 64;
    const int m = 8 * n + 2 * (at % 4) + i;
    const int64_t row = first + at / 4;
    float v[kUp ? 2 : 1];
#pragma unroll
    for (int k = 0; k < (kUp ? 2 : 1); ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) v[k] += part[p][n][2 * k + i][at];
    }
    if (m >= w.tokens || row >= w.rows) continue;
    if constexpr (kUp) {
      const float h = v[0] * gate(v[0], w.c0, w.c1) * v[1];
      const T upper = Traits<T>::store(h);
      const float rest = h - Traits<T>::load(upper);
      static_cast<T*>(w.out[0])[m * w.ldo + row] = upper;
      static_cast<T*>(w.out[1])[m * w.ldo + row] = Traits<T>::store(fabsf(rest) < INFINITY ? rest : 0.f);  // (infinity less itself)
    } else {
      static_cast<T*>(w.out[0])[m * w.ldo + row] = Traits<T>::store(v[0]);
    }
  }
}

// ---- fp32 ---------------------------------------------------------------------------------------------------
// Multiplications and additions: a warp has four rows of weights (two of either projection) and up to four tokens, a lane four numbers
// of each at a time; `share` warps of a block share the reduction, and neighbouring blocks have the next four tokens of the same rows.
// One token is bound by memory, 1024 x 2816 8.0 us, 2048 x 5632 27 (138 MB: 5.1 TB/s), 4096 x 10240 79 (6.4); more by the loads of
// tokens, 4 of them 14, 42 and 113 us, 8 20, 53 and 148.  Eight tokens a warp took 32, 78 and 224 (registers); three bf16 parts of each
// number and the matrix instructions 24, 59 and 185 of any up to 8, bound by taking the numbers apart, with 5 times the error.
constexpr int kWeights = 4, kLaneStep = 128;  // columns of a warp's step
template <bool kVec>
__device__ __forceinline__ float4 four(const float* row, int64_t at, int64_t depth) {
  if constexpr (kVec) {  // rows of whole and aligned runs of four
    const float4 v = *reinterpret_cast<const float4*>(row + (at < depth ? at : 0));
    return at < depth ? v : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  return make_float4(at < depth ? row[at] : 0.f, at + 1 < depth ? row[at + 1] : 0.f, at + 2 < depth ? row[at + 2] : 0.f, at + 3 < depth ? row[at + 3] : 0.f);
}
template <int kM, bool kUp, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) few32_kernel(const Few w, int share, int groups) {
  constexpr int kSet = kUp ? kWeights / 2 : kWeights, kAhead = 4, kSums = kWeights * kM;
  __shared__ float part[kWarps][kSums];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, slice = warp % share, sets = kWarps / share;
  const int token0 = static_cast<int>(blockIdx.x % groups) * kM;
  const int64_t first = static_cast<int64_t>(blockIdx.x / groups) * sets * kSet, row0 = first + warp / share * kSet;
  const float* weight[kWeights];
#pragma unroll
  for (int r = 0; r < kWeights; ++r) {
    const int64_t row = row0 + r % kSet;  // of rows that there are not, the first one
    weight[r] = static_cast<const float*>(w.w[r / kSet]) + (row < w.rows ? row : 0) * w.ldw[r / kSet];
  }
  const int64_t begin = slice * kLaneStep + lane * 4, step = share * kLaneStep;
  float4 run[kAhead][kWeights];
  auto load = [&](int64_t at) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int r = 0; r < kWeights; ++r) run[a][r] = four<kVec>(weight[r], at + a * step, w.depth);
  };
  if constexpr (!kUp) load(begin);  // as above
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if constexpr (kUp) load(begin);
  const float* token[kM];  // of tokens that there are not, the first one's
#pragma unroll
  for (int m = 0; m < kM; ++m) token[m] = static_cast<const float*>(w.x[0]) + (token0 + m < w.tokens ? token0 + m : 0) * w.ldx;
  float sum[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) sum[i] = 0.f;
  for (int64_t at = begin; at < w.depth; at += kAhead * step) {
    if (at != begin) load(at);
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int m = 0; m < kM; ++m) {
        const float4 x = four<kVec>(token[m], at + a * step, w.depth);
#pragma unroll
        for (int r = 0; r < kWeights; ++r) {
          float& v = sum[r * kM + m];
          v = fmaf(run[a][r].x, x.x, fmaf(run[a][r].y, x.y, fmaf(run[a][r].z, x.z, fmaf(run[a][r].w, x.w, v))));
        }
      }
  }
  // each lane hands on half of what it has, until it has one sum
#pragma unroll
  for (int o = 16, n = kSums; o > 0; o /= 2) {
    if (n > 1) {
      n /= 2;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float mine = lane & o ? sum[i + n] : sum[i], other = lane & o ? sum[i] : sum[i + n];
        sum[i] = mine + __shfl_xor_sync(0xFFFFFFFFu, other, o);
      }
    } else {
      sum[0] += __shfl_xor_sync(0xFFFFFFFFu, sum[0], o);
    }
  }
  if (lane % (32 / kSums) == 0) part[warp][lane / (32 / kSums)] = sum[0];
  __syncthreads();
  for (int item = threadIdx.x; item < sets * kSet * kM; item += kThreads) {
    const int m = item % kM, r = item / kM % kSet, set = item / (kM * kSet);
    const int64_t row = first + set * kSet + r;
    if (token0 + m >= w.tokens || row >= w.rows) continue;
    float v[2] = {0.f, 0.f};
    for (int p = set * share; p < (set + 1) * share; ++p) {
      v[0] += part[p][r * kM + m];
      if constexpr (kUp) v[1] += part[p][(kSet + r) * kM + m];
    }
    static_cast<float*>(w.out[0])[(token0 + m) * w.ldo + row] = kUp ? v[0] * gate_of(v[0], w.silu) * v[1] : v[0];
  }
}
// Warps that share a reduction: as many as leave the device full, and each a step.
template <bool kUp, bool kVec>
cudaError_t run32(const Few& w, cudaStream_t s) {
  constexpr int64_t kSet = kUp ? kWeights / 2 : kWeights, kFull = 148 * 16;
  const int64_t sets = (w.rows + kSet - 1) / kSet;
  int share = 1;
  while (share < kWarps && sets * share < kFull && w.depth > share * kLaneStep) share *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  const int groups = static_cast<int>((w.tokens + 3) / 4);
  cfg.gridDim = dim3(static_cast<unsigned>((sets * share + kWarps - 1) / kWarps * groups));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  if (w.tokens <= 1) return cudaLaunchKernelEx(&cfg, few32_kernel<1, kUp, kVec>, w, share, groups);
  if (w.tokens <= 2) return cudaLaunchKernelEx(&cfg, few32_kernel<2, kUp, kVec>, w, share, groups);
  return cudaLaunchKernelEx(&cfg, few32_kernel<4, kUp, kVec>, w, share, groups);
}

template <typename T, bool kUp, bool kVec>
cudaError_t run(const Few& w, cudaStream_t s) {
  if constexpr (std::is_same_v<T, float>) {
    return run32<kUp, kVec>(w, s);
  } else {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((w.rows + kRows - 1) / kRows));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  if (w.tokens <= 8) return cudaLaunchKernelEx(&cfg, few_kernel<T, 1, kUp, kVec>, w);
  if (w.tokens <= 16) return cudaLaunchKernelEx(&cfg, few_kernel<T, 2, kUp, kVec>, w);
  return cudaLaunchKernelEx(&cfg, few_kernel<T, 4, kUp, kVec>, w);
  }
}
template <typename T>
bool aligned(const GatedOperand& m, int64_t rows) {
  return reinterpret_cast<uintptr_t>(m.data) % 16 == 0 && (rows <= 1 || m.ld * sizeof(T) % 16 == 0);
}

template <typename T>
cudaError_t both(const GatedFew& g, cudaStream_t s) {
  const GatedShape& h = g.shape;
  const double log2e = 1.4426950408889634, gelu = 1.5957691216057308;  // 2 sqrt(2 / pi)
  const int64_t pitch = gated_pitch(h.hidden);
  constexpr int kRun = 16 / sizeof(T);
  T* const parts[2] = {static_cast<T*>(g.h), static_cast<T*>(g.h) + h.tokens * pitch};  // (fp32: the first alone)
  Few w{};
  w.c0 = static_cast<float>(h.activation == GatedActivation::kSilu ? -log2e : -log2e * gelu);
  w.silu = h.activation == GatedActivation::kSilu;
  w.c1 = h.activation == GatedActivation::kSilu ? 0.f : static_cast<float>(-log2e * gelu * 0.044715);
  w.tokens = static_cast<int>(h.tokens);
  w.x[0] = g.x.data;
  w.ldx = g.x.ld;
  w.w[0] = g.w_gate.data;
  w.w[1] = g.w_up.data;
  w.ldw[0] = g.w_gate.ld;
  w.ldw[1] = g.w_up.ld;
  w.out[0] = parts[0];
  w.out[1] = parts[1];
  w.ldo = pitch;
  w.rows = h.hidden;
  w.depth = h.width;
  const bool whole = h.width % kRun == 0 && aligned<T>(g.x, h.tokens) && aligned<T>(g.w_gate, h.hidden) && aligned<T>(g.w_up, h.hidden);
  const cudaError_t e = whole ? run<T, true, true>(w, s) : run<T, true, false>(w, s);
  if (e != cudaSuccess) return e;
  w.x[0] = parts[0];
  w.x[1] = parts[1];
  w.ldx = pitch;
  w.w[0] = g.w_down.data;
  w.ldw[0] = g.w_down.ld;
  w.out[0] = g.y;
  w.ldo = h.width;
  w.rows = h.width;
  w.depth = h.hidden;
  return h.hidden % kRun == 0 && aligned<T>(g.w_down, h.width) ? run<T, false, true>(w, s) : run<T, false, false>(w, s);
}

}  // namespace

cudaError_t launch_gated_few(const GatedFew& g, cudaStream_t s) {
  const GatedShape& h = g.shape;
  if (h.tokens <= 0 || h.tokens > kFewTokens || h.width <= 0 || h.hidden <= 0 || reinterpret_cast<uintptr_t>(g.h) % 16 != 0) return cudaErrorInvalidValue;
  if (h.width > 0x7FFFFFFFll || h.hidden > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  return g.f32 ? both<float>(g, s) : h.bf16 ? both<__nv_bfloat16>(g, s) : both<__half>(g, s);
}

}  // namespace kern
}  // namespace mccl
