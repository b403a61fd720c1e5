// Layer norm of rows, with the sum with a residual before it, and its gradients (sm_100a).
//
// Of a row s of n numbers: mean = sum(s) / n, rstd = 1 / sqrt(sum((s - mean)^2) / n + eps), u = (s - mean) rstd, y = u w + b.
// Backward, with g = dy w:
//     ds = rstd (g - mean(g) - u mean(g u)) + what else flows to s        dw = sum over rows of dy u        db = sum over rows of dy
// In fp32, each result rounded once.  The deviations are summed around the mean, from registers: a mean that is large against them costs nothing.
//
// Bound by memory: every number is read and written once.  A team of warps has a row in registers, and asks for the next one before it works on
// this one; blocks stay and go from row to row, so that weights are read once and, backward, a thread's columns and their sums for dw and db
// are its own.  These meet in shared memory at the end, and a second launch adds up the blocks', all in a fixed order.  Rows too long for that are
// read again from the second-level cache, and their columns summed by a launch of their own.
//
// us, bf16 with an fp32 residual, 8192 x 1024 (B200): forward 17 (96 MB: 5.5 TB/s), backward 25 (128 MB: 5.0) and 3 for the blocks' sums.  A row a
// block at a time, none asked for ahead, 25 and 38; a warp a row, 32 numbers a thread, 31 and 51; three blocks an SM 23 and 31.
// Rows that begin anywhere are read one number at a time: fp16, 4099 x 1723, 16 and 16 (with teams that just hold the row, 22 and 28: they make each
// address anew); bf16, 65535 x 17, 14 and 13 (61 and 41, of which 15 numbers of 16 a thread were none); 2048 x 8191 29 and 56.  Rows longer than 8192, which
// no team holds, bf16 with an fp32 residual, 2048 x 16384: 86 (4.7 TB/s), 122 and 39 for the columns.
#include "kernels/norm.cuh"

namespace mccl {
namespace kern {
namespace {

// kWarps: of a team, or 0 where it is told.
template <int kRun, int kN, int kWarps, typename X, typename S, typename Y, typename W>
__global__ void __launch_bounds__(kForwardThreads) norm_forward_kernel(const NormForward a, int told) {
  __shared__ float2 slots[2 * kForwardThreads / 32];
  const int warps = kWarps > 0 ? kWarps : told, team = 32 * warps, t = threadIdx.x % team, cols = a.shape.cols;
  const NormShape& h = a.shape;
  const X x_type(a.x.type);
  const S s_type(a.residual.type);
  const Y y_type(a.y_type);
  const W w_type(h.weight_type);
  const int teams = blockDim.x / team;
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  int64_t row = static_cast<int64_t>(blockIdx.x) * teams + threadIdx.x / team;
  if (row >= h.rows) return;  // a whole team
  Team sums(slots, warps, blockDim.x / 32);
  Raw<kRun, kN> x, r, w, b;
  auto ask = [&](int64_t row) {
    if (row >= h.rows) return;
    int at = t;
    if (kWarps == 0) asm volatile("" : "+r"(at));  // addresses are made anew: kept over the loop, one for each run and array, they take the registers
    x.load(a.x.data, x_type, row * a.x.ld, at, team, cols);
    if (a.residual.data != nullptr) r.load(a.residual.data, s_type, row * a.residual.ld, at, team, cols);
  };
  ask(row);
  if (h.weight != nullptr) w.load(h.weight, w_type, 0, t, team, cols);
  if (h.bias != nullptr) b.load(h.bias, w_type, 0, t, team, cols);
  const float per = 1.f / static_cast<float>(cols);
  for (; row < h.rows; row += step) {
    Row<kRun, kN> s, other;
    int at = t;
    if (kWarps == 0) asm volatile("" : "+r"(at));
    s.take(x, x_type);
    if (a.residual.data != nullptr) {
      other.take(r, s_type);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) s.v[n][i] += other.v[n][i];
      s.round(s_type);
    }
    ask(row + step);
    if (a.residual.data != nullptr) s.store(a.sum, s_type, row * cols, at, team, cols);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) sum += s.v[n][i];
    const float mean = sums.sum(sum) * per;
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
    const float rstd = 1.f / sqrtf(sums.sum(square) * per + h.eps);
    if (a.mean != nullptr && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    if (h.weight != nullptr) other.take(w, w_type);
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) s.v[n][i] *= h.weight != nullptr ? rstd * other.v[n][i] : rstd;
    if (h.bias != nullptr) {
      other.take(b, w_type);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) s.v[n][i] += other.v[n][i];
    }
    s.store(a.y, y_type, row * cols, at, team, cols);
  }
}

// Rows that no team has room for: a block has one, kFew numbers a thread at a time, and reads it again from the second-level cache.
template <int kRun>
__global__ void __launch_bounds__(kWideThreads, 2) norm_forward_wide_kernel(const NormForward a) {
  constexpr int kN = kFew / kRun, kStep = kWideThreads * kFew;
  __shared__ float2 slots[2 * kWideThreads / 32];
  const int cols = a.shape.cols, t = threadIdx.x;
  Team sums(slots, kWideThreads / 32, kWideThreads / 32);
  const NormShape& h = a.shape;
  const bool with = a.residual.data != nullptr;
  const Told x_type(a.x.type), s_type(with ? a.residual.type : a.x.type), y_type(a.y_type), w_type(h.weight_type);
  const void* const from = with ? a.sum : a.x.data;
  for (int64_t row = blockIdx.x; row < h.rows; row += gridDim.x) {
    const int64_t at = row * (with ? cols : a.x.ld);
    float sum = 0.f;
    for (int c = 0; c < cols; c += kStep) {
      Raw<kRun, kN> x, r;
      Row<kRun, kN> s, other;
      x.load(a.x.data, x_type, row * a.x.ld + c, t, kWideThreads, cols - c);
      if (with) r.load(a.residual.data, s_type, row * a.residual.ld + c, t, kWideThreads, cols - c);
      s.take(x, x_type);
      if (with) {
        other.take(r, s_type);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < kRun; ++i) s.v[n][i] += other.v[n][i];
        s.round(s_type);
        s.store(a.sum, s_type, row * cols + c, t, kWideThreads, cols - c);  // read again by this thread alone
      }
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) sum += s.v[n][i];
    }
    const float mean = sums.sum(sum) / static_cast<float>(cols);
    float square = 0.f;
    for (int c = 0; c < cols; c += kStep) {
      Raw<kRun, kN> x;
      Row<kRun, kN> s;
      x.load(from, s_type, at + c, t, kWideThreads, cols - c);
      s.take(x, s_type);
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const bool there = (n * kWideThreads + t) * kRun < cols - c;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          const float d = s.v[n][i] - mean;
          square = fmaf(d, there ? d : 0.f, square);
        }
      }
    }
    const float rstd = 1.f / sqrtf(sums.sum(square) / static_cast<float>(cols) + h.eps);
    if (a.mean != nullptr && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int c = 0; c < cols; c += kStep) {
      Raw<kRun, kN> x, w, b;
      Row<kRun, kN> s, other;
      x.load(from, s_type, at + c, t, kWideThreads, cols - c);
      if (h.weight != nullptr) w.load(h.weight, w_type, c, t, kWideThreads, cols - c);
      if (h.bias != nullptr) b.load(h.bias, w_type, c, t, kWideThreads, cols - c);
      s.take(x, s_type);
      if (h.weight != nullptr) other.take(w, w_type);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) s.v[n][i] = (s.v[n][i] - mean) * (h.weight != nullptr ? rstd * other.v[n][i] : rstd);
      if (h.bias != nullptr) {
        other.take(b, w_type);
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int i = 0; i < kRun; ++i) s.v[n][i] += other.v[n][i];
      }
      s.store(a.y, y_type, row * cols + c, t, kWideThreads, cols - c);
    }
  }
}

constexpr int kBlockWarps = 8;  // of a block where a team has fewer

template <int kRun, int kN, int kWarps, typename X, typename S, typename Y, typename W>
void teams(const NormForward& a, cudaStream_t s, int warps, Types<X, S, Y, W>) {
  const int all = block_warps(warps, kBlockWarps);
  norm_forward_kernel<kRun, kN, kWarps, X, S, Y, W>
      <<<static_cast<unsigned>(std::min<int64_t>(ceil_div(a.shape.rows, all / warps), kForwardBlocks)), 32 * all, 0, s>>>(a, warps);
}
template <int kRun, typename X, typename S, typename Y, typename W>
cudaError_t forward(const NormForward& a, cudaStream_t s, Types<X, S, Y, W> types, std::integral_constant<int, kRun>) {
  const NormShape& h = a.shape;
  note_launch();
  if (h.cols > kMany * kForwardThreads) {
    norm_forward_wide_kernel<kRun><<<static_cast<unsigned>(std::min<int64_t>(h.rows, 4 * kSms)), kWideThreads, 0, s>>>(a);
  } else if constexpr (kRun == 1) {
    const cudaError_t e = with_team(h.cols, [&](auto warps, auto numbers) {
      teams<1, decltype(numbers)::value, decltype(warps)::value>(a, s, warps, types);
      return cudaSuccess;
    });
    if (e != cudaSuccess) return e;
  } else {
    const int warps = static_cast<int>(ceil_div(h.cols, 32 * kMany));
    // fewer rows than fill the device have more threads each
    if (h.rows * warps < 16 * kSms && h.cols <= kFew * kForwardThreads) teams<kRun, kFew / kRun, 0>(a, s, static_cast<int>(ceil_div(h.cols, 32 * kFew)), types);
    else teams<kRun, kMany / kRun, 0>(a, s, warps, types);
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm_forward(const NormForward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  if (h.cols <= 0 || h.cols > kNormMostCols || h.rows < 0 || h.rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (h.rows == 0) return cudaSuccess;
  const bool sum = a.residual.data != nullptr;
  Alignment l(h.cols);
  l.with(a.x.data, a.x.ld, a.x.type);
  l.with(a.residual.data, a.residual.ld, a.residual.type);
  l.with(a.sum, h.cols, a.residual.type);
  l.with(a.y, h.cols, a.y_type);
  l.with(h.weight, h.cols, h.weight_type);
  l.with(h.bias, h.cols, h.weight_type);
  return with_types(a.x.type, sum ? a.residual.type : a.x.type, a.y_type, h.weight != nullptr || h.bias != nullptr ? h.weight_type : Elem::kF32, [&](auto types) {
    return with_run(types, l.run, [&](auto t, auto run) { return forward(a, s, t, run); });
  });
}

}  // namespace kern
}  // namespace mccl
