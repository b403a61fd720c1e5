// Layer norm of rows, with the sum with a residual before it, and its gradients (sm_100a).
//
// Of a row s of n numbers: mean = sum(s) / n, rstd = 1 / sqrt(sum((s - mean)^2) / n + eps), u = (s - mean) rstd, y = u w + b.
// Backward, with g = dy w:
//     ds = rstd (g - mean(g) - u mean(g u)) + what else flows to s        dw = sum over rows of dy u        db = sum over rows of dy
// In fp32, each result rounded once.  The deviations are summed around the mean, from registers: a mean that is large against them costs nothing.
//
// Bound by memory: every number is read and written once.  A team of warps has a row in registers.  Backward, blocks stay and go from row to
// row, so that a thread's columns and their sums for dw and db stay its own; these meet in shared memory at the end, and a second launch adds
// up the blocks', all in a fixed order.  Rows too long for that are read twice, and the columns summed by a launch of their own.
#include <algorithm>

#include "kernels/elems.cuh"
#include "kernels/launch_count.h"
#include "kernels/norm_api.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kSms = 148;
constexpr int kFew = 8, kMore = 16, kMany = 32;              // numbers of a row that a thread has
constexpr int kForwardThreads = 512, kBackwardThreads = 512;  // of a block, at most
constexpr int kWideThreads = 512;
constexpr int kBackwardBlocks = 3 * kSms;                    // that stay

template <int kRun>
__device__ __forceinline__ void zero_run(float (&v)[kRun]) {
#pragma unroll
  for (int i = 0; i < kRun; ++i) v[i] = 0.f;
}
// kRun numbers that are aligned to their run's size (16 bytes at most).
template <int kRun>
__device__ __forceinline__ void get(const void* p, Elem type, int64_t at, float (&v)[kRun]) {
  if (type == Elem::kF32) load_run<float, kRun>(static_cast<const float*>(p) + at, kRun, true, v);
  else if (type == Elem::kBF16) load_run<__nv_bfloat16, kRun>(static_cast<const __nv_bfloat16*>(p) + at, kRun, true, v);
  else load_run<__half, kRun>(static_cast<const __half*>(p) + at, kRun, true, v);
}
template <int kRun>
__device__ __forceinline__ void put(void* p, Elem type, int64_t at, const float (&v)[kRun]) {
  if (type == Elem::kF32) store_run<float, kRun>(static_cast<float*>(p) + at, kRun, true, v);
  else if (type == Elem::kBF16) store_run<__nv_bfloat16, kRun>(static_cast<__nv_bfloat16*>(p) + at, kRun, true, v);
  else store_run<__half, kRun>(static_cast<__half*>(p) + at, kRun, true, v);
}
// A thread's runs of a row: every `team`th, so that neighbours have neighbouring runs.
template <int kRun, int kN>
struct Row {
  float v[kN][kRun];
  template <typename T>
  __device__ __forceinline__ void load(const T* p, int t, int team, int cols) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int c = (n * team + t) * kRun;
      if (c < cols) load_run<T, kRun>(p + c, kRun, true, v[n]);
      else zero_run(v[n]);
    }
  }
  // One by one, the types of 16 bits by one loop: three of them, with their addresses, took 240 registers.
  __device__ __forceinline__ void load_singly(const void* p, Elem type, int64_t at, int t, int team, int cols) {
    if (type == Elem::kF32) {
      load(static_cast<const float*>(p) + at, t, team, cols);
    } else {
      const uint16_t* f = static_cast<const uint16_t*>(p) + at;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int c = n * team + t;
        const uint16_t x = c < cols ? f[c] : uint16_t{0};
        v[n][0] = type == Elem::kBF16 ? __uint_as_float(static_cast<uint32_t>(x) << 16) : __half2float(__ushort_as_half(x));
      }
    }
  }
  __device__ __forceinline__ void store_singly(void* p, Elem type, int64_t at, int t, int team, int cols) const {
    if (type == Elem::kF32) {
      store(static_cast<float*>(p) + at, t, team, cols);
    } else {
      uint16_t* f = static_cast<uint16_t*>(p) + at;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int c = n * team + t;
        const uint16_t x = type == Elem::kBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[n][0])) : __half_as_ushort(__float2half_rn(v[n][0]));
        if (c < cols) f[c] = x;
      }
    }
  }
  __device__ __forceinline__ void load(const void* p, Elem type, int64_t at, int t, int team, int cols) {
    if constexpr (kRun == 1) {
      load_singly(p, type, at, t, team, cols);
      return;
    }
    if (type == Elem::kF32) load(static_cast<const float*>(p) + at, t, team, cols);
    else if (type == Elem::kBF16) load(static_cast<const __nv_bfloat16*>(p) + at, t, team, cols);
    else load(static_cast<const __half*>(p) + at, t, team, cols);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p, int t, int team, int cols) const {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int c = (n * team + t) * kRun;
      if (c < cols) store_run<T, kRun>(p + c, kRun, true, v[n]);
    }
  }
  __device__ __forceinline__ void store(void* p, Elem type, int64_t at, int t, int team, int cols) const {
    if constexpr (kRun == 1) {
      store_singly(p, type, at, t, team, cols);
      return;
    }
    if (type == Elem::kF32) store(static_cast<float*>(p) + at, t, team, cols);
    else if (type == Elem::kBF16) store(static_cast<__nv_bfloat16*>(p) + at, t, team, cols);
    else store(static_cast<__half*>(p) + at, t, team, cols);
  }
  // As the type keeps it.
  __device__ __forceinline__ void round(Elem type) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        v[n][i] = type == Elem::kBF16 ? __bfloat162float(__float2bfloat16_rn(v[n][i])) : type == Elem::kF16 ? __half2float(__float2half_rn(v[n][i])) : v[n][i];
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
  __device__ __forceinline__ float sum(float a) { return sum(a, 0.f).x; }
};

template <int kRun, int kN>
__global__ void __launch_bounds__(kForwardThreads) norm_forward_kernel(const NormForward a, int warps) {
  __shared__ float2 slots[2 * kForwardThreads / 32];
  const int team = 32 * warps, t = threadIdx.x % team, cols = a.shape.cols;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / team) + threadIdx.x / team;
  if (row >= a.shape.rows) return;  // a whole team
  Team sums(slots, warps, blockDim.x / 32);
  Row<kRun, kN> s;
  s.load(a.x.data, a.x.type, row * a.x.ld, t, team, cols);
  if (a.residual.data != nullptr) {
    Row<kRun, kN> r;
    r.load(a.residual.data, a.residual.type, row * a.residual.ld, t, team, cols);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) s.v[n][i] += r.v[n][i];
    s.round(a.residual.type);
    s.store(a.sum, a.residual.type, row * cols, t, team, cols);
  }
  float sum = 0.f;
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int i = 0; i < kRun; ++i) sum += s.v[n][i];
  const float mean = sums.sum(sum) / static_cast<float>(cols);
  float square = 0.f;
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const bool there = (n * team + t) * kRun < cols;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      s.v[n][i] -= mean;
      square = fmaf(s.v[n][i], there ? s.v[n][i] : 0.f, square);
    }
  }
  const float rstd = 1.f / sqrtf(sums.sum(square) / static_cast<float>(cols) + a.shape.eps);
  if (a.mean != nullptr && t == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const NormShape& h = a.shape;
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int c = (n * team + t) * kRun;
    if (c >= cols) continue;
    float w[kRun], b[kRun];
    if (h.weight != nullptr) get<kRun>(h.weight, h.weight_type, c, w);
    if (h.bias != nullptr) get<kRun>(h.bias, h.weight_type, c, b);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      float y = s.v[n][i] * rstd;
      if (h.weight != nullptr) y *= w[i];
      if (h.bias != nullptr) y += b[i];
      s.v[n][i] = y;
    }
  }
  s.store(a.y, a.y_type, row * cols, t, team, cols);
}

// Rows that no team has room for: a block has one, and reads it again from the second-level cache.
template <int kRun>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const NormForward a) {
  __shared__ float2 slots[2 * kWideThreads / 32];
  const int cols = a.shape.cols, step = kWideThreads * kRun;
  Team sums(slots, kWideThreads / 32, kWideThreads / 32);
  const NormShape& h = a.shape;
  for (int64_t row = blockIdx.x; row < h.rows; row += gridDim.x) {
    float sum = 0.f;
    for (int c = threadIdx.x * kRun; c < cols; c += step) {
      float v[kRun];
      get<kRun>(a.x.data, a.x.type, row * a.x.ld + c, v);
      if (a.residual.data != nullptr) {
        float r[kRun];
        get<kRun>(a.residual.data, a.residual.type, row * a.residual.ld + c, r);
#pragma unroll
        for (int i = 0; i < kRun; ++i) v[i] += r[i];
        put<kRun>(a.sum, a.residual.type, row * cols + c, v);
        get<kRun>(a.sum, a.residual.type, row * cols + c, v);  // this thread's own: what was kept
      }
#pragma unroll
      for (int i = 0; i < kRun; ++i) sum += v[i];
    }
    const void* from = a.residual.data != nullptr ? a.sum : a.x.data;
    const Elem type = a.residual.data != nullptr ? a.residual.type : a.x.type;
    const int64_t at = row * (a.residual.data != nullptr ? cols : a.x.ld);
    const float mean = sums.sum(sum) / static_cast<float>(cols);
    float square = 0.f;
    for (int c = threadIdx.x * kRun; c < cols; c += step) {
      float v[kRun];
      get<kRun>(from, type, at + c, v);
#pragma unroll
      for (int i = 0; i < kRun; ++i) square = fmaf(v[i] - mean, v[i] - mean, square);
    }
    const float rstd = 1.f / sqrtf(sums.sum(square) / static_cast<float>(cols) + h.eps);
    if (a.mean != nullptr && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int c = threadIdx.x * kRun; c < cols; c += step) {
      float v[kRun], w[kRun], b[kRun];
      get<kRun>(from, type, at + c, v);
      if (h.weight != nullptr) get<kRun>(h.weight, h.weight_type, c, w);
      if (h.bias != nullptr) get<kRun>(h.bias, h.weight_type, c, b);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        v[i] = (v[i] - mean) * rstd;
        if (h.weight != nullptr) v[i] *= w[i];
        if (h.bias != nullptr) v[i] += b[i];
      }
      put<kRun>(a.y, a.y_type, row * cols + c, v);
    }
  }
}

// ---- backward -------------------------------------------------------------------------------------------------
template <int kRun, int kN>
__global__ void __launch_bounds__(kBackwardThreads) norm_backward_kernel(const NormBackward a, int warps) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 slots[2 * kBackwardThreads / 32];
  extern __shared__ float columns[];  // [2][cols]
  const NormShape& h = a.shape;
  const int team = 32 * warps, t = threadIdx.x % team, cols = h.cols, teams = blockDim.x / team, number = threadIdx.x / team;
  Team sums(slots, warps, blockDim.x / 32);
  Row<kRun, kN> w;
  if (h.weight != nullptr) {
    w.load(h.weight, h.weight_type, 0, t, team, cols);
  } else {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) w.v[n][i] = 1.f;
  }
  float dw[kN][kRun], db[kN][kRun];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    zero_run(dw[n]);
    zero_run(db[n]);
  }
  const float per = 1.f / static_cast<float>(cols);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * teams + number; row < h.rows; row += static_cast<int64_t>(gridDim.x) * teams) {
    int at = t;
    asm volatile("" : "+r"(at));  // addresses are made anew: kept over the loop, one for each run and array, they take all registers
    Row<kRun, kN> s, g;
    s.load(a.s.data, a.s.type, row * a.s.ld, at, team, cols);
    g.load(a.dy.data, a.dy.type, row * a.dy.ld, at, team, cols);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float first = 0.f, second = 0.f;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {  // (beyond the row dy is zero, and with it all of these)
        const float u = (s.v[n][i] - mean) * rstd, dy = g.v[n][i];
        dw[n][i] = fmaf(dy, u, dw[n][i]);
        db[n][i] += dy;
        s.v[n][i] = u;
        g.v[n][i] = dy * w.v[n][i];
        first += g.v[n][i];
        second = fmaf(g.v[n][i], u, second);
      }
    if (a.dx == nullptr && a.dresidual == nullptr) continue;
    Row<kRun, kN> ds;
    if (a.ds.data != nullptr) ds.load(a.ds.data, a.ds.type, row * a.ds.ld, at, team, cols);
    const float2 both = sums.sum(first, second);
    const float c1 = both.x * per, c2 = both.y * per;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        g.v[n][i] = rstd * (g.v[n][i] - c1 - s.v[n][i] * c2);
        if (a.ds.data != nullptr) g.v[n][i] += ds.v[n][i];
      }
    if (a.dx != nullptr) g.store(a.dx, a.dx_type, row * cols, at, team, cols);
    if (a.dresidual != nullptr) g.store(a.dresidual, a.s.type, row * cols, at, team, cols);
  }
  if (a.partial == nullptr) return;
  for (int turn = 0; turn < teams; ++turn) {  // one team behind the other, so that the order is always the same
    if (number == turn) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int c = (n * team + t) * kRun;
        if (c >= cols) continue;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          columns[c + i] = (turn ? columns[c + i] : 0.f) + dw[n][i];
          columns[cols + c + i] = (turn ? columns[cols + c + i] : 0.f) + db[n][i];
        }
      }
    }
    __syncthreads();
  }
  float* to = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
  for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) to[i] = columns[i];
}
template <int kRun>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(const NormBackward a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 slots[2 * kWideThreads / 32];
  const NormShape& h = a.shape;
  const int cols = h.cols, step = kWideThreads * kRun;
  Team sums(slots, kWideThreads / 32, kWideThreads / 32);
  const float per = 1.f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < h.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float u[kRun], g[kRun];
    auto both_of = [&](int c) {
      float w[kRun];
      get<kRun>(a.s.data, a.s.type, row * a.s.ld + c, u);
      get<kRun>(a.dy.data, a.dy.type, row * a.dy.ld + c, g);
      if (h.weight != nullptr) get<kRun>(h.weight, h.weight_type, c, w);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        u[i] = (u[i] - mean) * rstd;
        if (h.weight != nullptr) g[i] *= w[i];
      }
    };
    float first = 0.f, second = 0.f;
    for (int c = threadIdx.x * kRun; c < cols; c += step) {
      both_of(c);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        first += g[i];
        second = fmaf(g[i], u[i], second);
      }
    }
    const float2 both = sums.sum(first, second);
    const float c1 = both.x * per, c2 = both.y * per;
    for (int c = threadIdx.x * kRun; c < cols; c += step) {
      both_of(c);
      float ds[kRun];
      if (a.ds.data != nullptr) get<kRun>(a.ds.data, a.ds.type, row * a.ds.ld + c, ds);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        g[i] = rstd * (g[i] - c1 - u[i] * c2);
        if (a.ds.data != nullptr) g[i] += ds[i];
      }
      if (a.dx != nullptr) put<kRun>(a.dx, a.dx_type, row * cols + c, g);
      if (a.dresidual != nullptr) put<kRun>(a.dresidual, a.s.type, row * cols + c, g);
    }
  }
}
// The columns' sums over some of the rows, a column a thread, for rows that are too long for the kernel above.
constexpr int kColumnThreads = 256;
__global__ void __launch_bounds__(kColumnThreads) norm_columns_kernel(const NormBackward a, int64_t rows_each) {
  const int c = blockIdx.x * kColumnThreads + threadIdx.x, cols = a.shape.cols;
  if (c >= cols) return;
  const int64_t begin = blockIdx.y * rows_each, end = min(a.shape.rows, begin + rows_each);
  float dw = 0.f, db = 0.f;
#pragma unroll 4
  for (int64_t row = begin; row < end; ++row) {
    float s[1], dy[1];
    get<1>(a.s.data, a.s.type, row * a.s.ld + c, s);
    get<1>(a.dy.data, a.dy.type, row * a.dy.ld + c, dy);
    dw = fmaf(dy[0], (s[0] - a.mean[row]) * a.rstd[row], dw);
    db += dy[0];
  }
  float* to = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * cols;
  to[c] = dw;
  to[cols + c] = db;
}
// Adds up the blocks' sums: 32 columns a block, whose warps share the parts.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(const float* partial, int parts, int cols, void* dweight, void* dbias, Elem type) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kWarps = kJoinThreads / 32;
  __shared__ float sums[kWarps][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane, all = 2ll * cols;
  float sum = 0.f;
  if (c < all)
#pragma unroll 8
    for (int p = warp; p < parts; p += kWarps) sum += __ldcg(partial + p * all + c);
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp > 0 || c >= all) return;
  for (int i = 1; i < kWarps; ++i) sum += sums[i][lane];
  void* to = c < cols ? dweight : dbias;
  const float v[1] = {sum};
  if (to != nullptr) put<1>(to, type, c < cols ? c : c - cols, v);
}

// ---- host ---------------------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int size_of(Elem e) { return e == Elem::kF32 ? 4 : 2; }

// The longest run that all arrays are aligned to: 8 numbers of 16 bits, 4 beside numbers of 32, or one.
struct Alignment {
  int run;
  explicit Alignment(int cols) : run(cols % 8 == 0 ? 8 : cols % 4 == 0 ? 4 : 1) {}
  void with(const void* p, int64_t ld, Elem type) {
    if (p == nullptr) return;
    if (type == Elem::kF32) run = std::min(run, 4);
    while (run > 1 && (reinterpret_cast<uintptr_t>(p) % (run * size_of(type)) != 0 || ld % run != 0)) run = run == 8 ? 4 : 1;
  }
};

int block_warps(int warps, int most) { return warps * std::max(1, most / warps); }

constexpr int kForwardWarps = 8, kBackwardWarps = 8;  // of a block where a team has fewer

bool backward_wide(const NormShape& s) { return s.cols > kMore * kBackwardThreads; }
// Warps of a backward team.
int backward_warps(const NormShape& s) { return static_cast<int>(ceil_div(s.cols, 32 * (s.cols <= kFew * kBackwardThreads ? kFew : kMore))); }
// Blocks of the backward kernel, or parts of the rows for the columns' sums.
int parts_of(const NormShape& s) {
  if (backward_wide(s)) return static_cast<int>(std::clamp<int64_t>(ceil_div(8 * kSms, ceil_div(s.cols, kColumnThreads)), 1, ceil_div(s.rows, 16)));
  const int warps = backward_warps(s), teams = block_warps(warps, kBackwardWarps) / warps;
  return static_cast<int>(std::min<int64_t>(ceil_div(s.rows, teams), kBackwardBlocks));
}

template <int kRun>
cudaError_t forward(const NormForward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  note_launch();
  int warps = static_cast<int>(ceil_div(h.cols, 32 * kMany));
  // fewer rows than fill the device have more threads each
  if (h.rows * warps < 16 * kSms && h.cols <= kFew * kForwardThreads) {
    warps = static_cast<int>(ceil_div(h.cols, 32 * kFew));
    const int all = block_warps(warps, kForwardWarps);
    norm_forward_kernel<kRun, kFew / kRun><<<static_cast<unsigned>(ceil_div(h.rows, all / warps)), 32 * all, 0, s>>>(a, warps);
  } else if (h.cols <= kMany * kForwardThreads) {
    const int all = block_warps(warps, kForwardWarps);
    norm_forward_kernel<kRun, kMany / kRun><<<static_cast<unsigned>(ceil_div(h.rows, all / warps)), 32 * all, 0, s>>>(a, warps);
  } else {
    norm_forward_wide_kernel<kRun><<<static_cast<unsigned>(std::min<int64_t>(h.rows, 4 * kSms)), kWideThreads, 0, s>>>(a);
  }
  return cudaGetLastError();
}

template <int kRun>
cudaError_t backward(const NormBackward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  const int parts = parts_of(h);
  if (backward_wide(h)) {
    if (a.dx != nullptr || a.dresidual != nullptr) {
      note_launch();
      norm_backward_wide_kernel<kRun><<<static_cast<unsigned>(std::min<int64_t>(h.rows, 4 * kSms)), kWideThreads, 0, s>>>(a);
    }
    if (a.partial != nullptr) {
      note_launch();
      const int64_t each = ceil_div(h.rows, parts);
      norm_columns_kernel<<<dim3(static_cast<unsigned>(ceil_div(h.cols, kColumnThreads)), parts), kColumnThreads, 0, s>>>(a, each);
    }
  } else {
    const int warps = backward_warps(h), all = block_warps(warps, kBackwardWarps), shared = 2 * h.cols * 4;
    const auto kernel = h.cols <= kFew * kBackwardThreads ? norm_backward_kernel<kRun, kFew / kRun> : norm_backward_kernel<kRun, kMore / kRun>;
    if (shared > 40 * 1024) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMore * kBackwardThreads * 4);
      if (e != cudaSuccess) return e;
    }
    note_launch();
    kernel<<<parts, 32 * all, shared, s>>>(a, warps);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || a.partial == nullptr) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div(2ll * h.cols, 32)));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, norm_join_kernel, static_cast<const float*>(a.partial), parts, h.cols, a.dweight, a.dbias, h.weight_type);
}

}  // namespace

cudaError_t launch_norm_forward(const NormForward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  if (h.cols <= 0 || h.rows < 0 || h.rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (h.rows == 0) return cudaSuccess;
  Alignment l(h.cols);
  l.with(a.x.data, a.x.ld, a.x.type);
  l.with(a.residual.data, a.residual.ld, a.residual.type);
  l.with(a.sum, h.cols, a.residual.type);
  l.with(a.y, h.cols, a.y_type);
  l.with(h.weight, h.cols, h.weight_type);
  l.with(h.bias, h.cols, h.weight_type);
  return l.run == 8 ? forward<8>(a, s) : l.run == 4 ? forward<4>(a, s) : forward<1>(a, s);
}

int64_t norm_partial_bytes(const NormShape& s) { return s.rows <= 0 ? 0 : static_cast<int64_t>(parts_of(s)) * 2 * s.cols * 4; }

cudaError_t launch_norm_backward(const NormBackward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  if (h.cols <= 0 || h.rows < 0 || h.rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (h.rows == 0) return cudaSuccess;
  Alignment l(h.cols);
  l.with(a.s.data, a.s.ld, a.s.type);
  l.with(a.dy.data, a.dy.ld, a.dy.type);
  l.with(a.ds.data, a.ds.ld, a.ds.type);
  l.with(a.dx, h.cols, a.dx_type);
  l.with(a.dresidual, h.cols, a.s.type);
  l.with(h.weight, h.cols, h.weight_type);
  return l.run == 8 ? backward<8>(a, s) : l.run == 4 ? backward<4>(a, s) : backward<1>(a, s);
}

}  // namespace kern
}  // namespace mccl
