// Gradients of layer norm (see norm_forward.cu for the formulas).
#include "kernels/norm.cuh"

namespace mccl {
namespace kern {
namespace {

// kWarps: of a team, or 0 where it is told.
template <int kRun, int kN, int kWarps, typename X, typename S, typename Y, typename W>
__global__ void __launch_bounds__(kBackwardThreads) norm_backward_kernel(const NormBackward a, int told) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float2 slots[2 * kBackwardThreads / 32];
  extern __shared__ float columns[];  // [2][cols]
  const NormShape& h = a.shape;
  const X x_type(a.dx_type);
  const S s_type(a.s.type);
  const Y y_type(a.dy.type);
  const W w_type(h.weight_type);
  const int warps = kWarps > 0 ? kWarps : told, team = 32 * warps, t = threadIdx.x % team, cols = h.cols, teams = blockDim.x / team, number = threadIdx.x / team;
  Team sums(slots, warps, blockDim.x / 32);
  Row<kRun, kN> w;
  w.fill(1.f);
  if (h.weight != nullptr) {
    Raw<kRun, kN> raw;
    raw.load(h.weight, w_type, 0, t, team, cols);
    w.take(raw, w_type);
  }
  Row<kRun, kN> dw, db;
  dw.fill(0.f);
  db.fill(0.f);
  const float per = 1.f / static_cast<float>(cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  Raw<kRun, kN> next_s, next_g, next_ds;
  float next_mean = 0.f, next_rstd = 0.f;
  auto ask = [&](int64_t row) {
    if (row >= h.rows) return;
    int at = t;
    if (kWarps == 0) asm volatile("" : "+r"(at));  // addresses are made anew: kept over the loop, one for each run and array, they take all registers
    next_s.load(a.s.data, s_type, row * a.s.ld, at, team, cols);
    next_g.load(a.dy.data, y_type, row * a.dy.ld, at, team, cols);
    if (a.ds.data != nullptr) next_ds.load(a.ds.data, s_type, row * a.ds.ld, at, team, cols);
    next_mean = a.mean[row];
    next_rstd = a.rstd[row];
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * teams + number;
  constexpr bool kAhead = kRun * kN <= 8;  // the next row is asked for before this one is worked on; of longer ones there is no room for it
  if (kAhead) ask(row);
  for (; row < h.rows; row += step) {
    if (!kAhead) ask(row);
    Row<kRun, kN> s, g, ds;
    s.take(next_s, s_type);
    g.take(next_g, y_type);
    if (a.ds.data != nullptr) ds.take(next_ds, s_type);
    const float mean = next_mean, rstd = next_rstd;
    if (kAhead) ask(row + step);
    float first = 0.f, second = 0.f;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {  // (beyond the row dy is zero, and with it all of these)
        const float u = (s.v[n][i] - mean) * rstd, dy = g.v[n][i];
        dw.v[n][i] = fmaf(dy, u, dw.v[n][i]);
        db.v[n][i] += dy;
        s.v[n][i] = u;
        g.v[n][i] = dy * w.v[n][i];
        first += g.v[n][i];
        second = fmaf(g.v[n][i], u, second);
      }
    if (a.dx == nullptr && a.dresidual == nullptr) continue;
    const float2 both = sums.sum(first, second);
    const float c1 = both.x * per, c2 = both.y * per;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        g.v[n][i] = rstd * (g.v[n][i] - c1 - s.v[n][i] * c2);
        if (a.ds.data != nullptr) g.v[n][i] += ds.v[n][i];
      }
    int at = t;
    if (kWarps == 0) asm volatile("" : "+r"(at));
    if (a.dx != nullptr) g.store(a.dx, x_type, row * cols, at, team, cols);
    if (a.dresidual != nullptr) g.store(a.dresidual, s_type, row * cols, at, team, cols);
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
          columns[c + i] = (turn ? columns[c + i] : 0.f) + dw.v[n][i];
          columns[cols + c + i] = (turn ? columns[cols + c + i] : 0.f) + db.v[n][i];
        }
      }
    }
    __syncthreads();
  }
  float* to = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
  for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) to[i] = columns[i];
}
// Rows that no team has room for: a run, or kFew numbers, a thread at a time, read again from the second-level cache.
template <int kRun>
__global__ void __launch_bounds__(kWideThreads, 2) norm_backward_wide_kernel(const NormBackward a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int kN = kRun == 1 ? kFew : 1, kStep = kWideThreads * kRun * kN;
  __shared__ float2 slots[2 * kWideThreads / 32];
  const NormShape& h = a.shape;
  const int cols = h.cols, t = threadIdx.x;
  Team sums(slots, kWideThreads / 32, kWideThreads / 32);
  const Told x_type(a.dx_type), s_type(a.s.type), y_type(a.dy.type), w_type(h.weight_type);
  const float per = 1.f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < h.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    Row<kRun, kN> u, g;
    auto both_of = [&](int c) {
      Raw<kRun, kN> s, dy, w;
      s.load(a.s.data, s_type, row * a.s.ld + c, t, kWideThreads, cols - c);
      dy.load(a.dy.data, y_type, row * a.dy.ld + c, t, kWideThreads, cols - c);
      if (h.weight != nullptr) w.load(h.weight, w_type, c, t, kWideThreads, cols - c);
      u.take(s, s_type);
      g.take(dy, y_type);
      Row<kRun, kN> weight;
      weight.fill(1.f);
      if (h.weight != nullptr) weight.take(w, w_type);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          u.v[n][i] = (u.v[n][i] - mean) * rstd;
          g.v[n][i] *= weight.v[n][i];
        }
    };
    float first = 0.f, second = 0.f;
    for (int c = 0; c < cols; c += kStep) {
      both_of(c);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) {  // (beyond the row dy is zero, and with it these)
          first += g.v[n][i];
          second = fmaf(g.v[n][i], u.v[n][i], second);
        }
    }
    const float2 both = sums.sum(first, second);
    const float c1 = both.x * per, c2 = both.y * per;
    for (int c = 0; c < cols; c += kStep) {
      Raw<kRun, kN> more;
      if (a.ds.data != nullptr) more.load(a.ds.data, s_type, row * a.ds.ld + c, t, kWideThreads, cols - c);
      both_of(c);
      Row<kRun, kN> ds;
      ds.fill(0.f);
      if (a.ds.data != nullptr) ds.take(more, s_type);
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < kRun; ++i) g.v[n][i] = rstd * (g.v[n][i] - c1 - u.v[n][i] * c2) + ds.v[n][i];
      if (a.dx != nullptr) g.store(a.dx, x_type, row * cols + c, t, kWideThreads, cols - c);
      if (a.dresidual != nullptr) g.store(a.dresidual, s_type, row * cols + c, t, kWideThreads, cols - c);
    }
  }
}
// The columns' sums over some of the rows, a run of columns a thread, for rows that are too long for the kernel above.
constexpr int kColumnThreads = 256, kRowsAhead = 4;
template <int kRun>
__global__ void __launch_bounds__(kColumnThreads) norm_columns_kernel(const NormBackward a, int64_t rows_each) {
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * kColumnThreads + threadIdx.x) * kRun;
  const int cols = a.shape.cols;
  if (c >= cols) return;
  const Told s_type(a.s.type), y_type(a.dy.type);
  const int64_t begin = blockIdx.y * rows_each, end = min(a.shape.rows, begin + rows_each);
  float dw[kRun], db[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) dw[i] = db[i] = 0.f;
  for (int64_t row = begin; row < end; row += kRowsAhead) {
    Raw<kRun, 1> s[kRowsAhead], dy[kRowsAhead];
    float mean[kRowsAhead], rstd[kRowsAhead];
#pragma unroll
    for (int r = 0; r < kRowsAhead; ++r) {
      const int64_t at = min(row + r, end - 1);
      s[r].load(a.s.data, s_type, at * a.s.ld + c, 0, 1, kRun);
      dy[r].load(a.dy.data, y_type, at * a.dy.ld + c, 0, 1, kRun);
      mean[r] = a.mean[at];
      rstd[r] = a.rstd[at];
    }
#pragma unroll
    for (int r = 0; r < kRowsAhead; ++r) {
      if (row + r >= end) break;
      Row<kRun, 1> u, g;
      u.take(s[r], s_type);
      g.take(dy[r], y_type);
#pragma unroll
      for (int i = 0; i < kRun; ++i) {
        dw[i] = fmaf(g.v[0][i], (u.v[0][i] - mean[r]) * rstd[r], dw[i]);
        db[i] += g.v[0][i];
      }
    }
  }
  float* to = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * cols;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    to[c + i] = dw[i];
    to[cols + c + i] = db[i];
  }
}
// Adds up the blocks' sums: 32 columns a block, whose warps share the parts.
constexpr int kJoinThreads = 1024;
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
constexpr int kBlockWarps = 8;  // of a block where a team has fewer
bool backward_wide(const NormShape& s) { return s.cols > kMany * kBackwardThreads; }
// Parts of the rows for the columns' sums of long ones, by runs of `run`.
int parts_of(const NormShape& s, int run) { return static_cast<int>(std::clamp<int64_t>(ceil_div(8 * kSms, ceil_div(s.cols, run * kColumnThreads)), 1, ceil_div(s.rows, 16))); }

// Its blocks.
template <int kRun, int kN, int kWarps, typename X, typename S, typename Y, typename W>
cudaError_t teams(const NormBackward& a, cudaStream_t s, int warps, Types<X, S, Y, W>, int* blocks) {
  const NormShape& h = a.shape;
  const int all = block_warps(warps, kBlockWarps), shared = 2 * h.cols * 4;
  const auto kernel = norm_backward_kernel<kRun, kN, kWarps, X, S, Y, W>;
  if (shared > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMany * kBackwardThreads * 4);
    if (e != cudaSuccess) return e;
  }
  *blocks = static_cast<int>(std::min<int64_t>(ceil_div(h.rows, all / warps), kBackwardBlocks));
  note_launch();
  kernel<<<*blocks, 32 * all, shared, s>>>(a, warps);
  return cudaGetLastError();
}
template <int kRun, typename X, typename S, typename Y, typename W>
cudaError_t backward(const NormBackward& a, cudaStream_t s, Types<X, S, Y, W> types, std::integral_constant<int, kRun>) {
  const NormShape& h = a.shape;
  int parts = 0;
  if (backward_wide(h)) {
    parts = parts_of(h, kRun);
    if (a.dx != nullptr || a.dresidual != nullptr) {
      note_launch();
      norm_backward_wide_kernel<kRun><<<static_cast<unsigned>(std::min<int64_t>(h.rows, 4 * kSms)), kWideThreads, 0, s>>>(a);
    }
    if (a.partial != nullptr) {
      note_launch();
      const int64_t each = ceil_div(h.rows, parts);
      norm_columns_kernel<kRun><<<dim3(static_cast<unsigned>(ceil_div(h.cols, kRun * kColumnThreads)), parts), kColumnThreads, 0, s>>>(a, each);
    }
  } else {
    cudaError_t e;
    if constexpr (kRun == 1)
      e = with_team(h.cols, [&](auto warps, auto numbers) { return teams<1, decltype(numbers)::value, decltype(warps)::value>(a, s, warps, types, &parts); });
    else if (h.cols <= kFew * kBackwardThreads)
      e = teams<kRun, kFew / kRun, 0>(a, s, static_cast<int>(ceil_div(h.cols, 32 * kFew)), types, &parts);
    else
      e = teams<kRun, kMany / kRun, 0>(a, s, static_cast<int>(ceil_div(h.cols, 32 * kMany)), types, &parts);
    if (e != cudaSuccess) return e;
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

// (as many as there may be, whatever the rows are aligned to)
int64_t norm_partial_bytes(const NormShape& s) {
  if (s.rows <= 0) return 0;
  return (backward_wide(s) ? parts_of(s, 8) : std::min<int64_t>(s.rows, kBackwardBlocks)) * 2 * s.cols * 4;
}

cudaError_t launch_norm_backward(const NormBackward& a, cudaStream_t s) {
  const NormShape& h = a.shape;
  if (h.cols <= 0 || h.cols > kNormMostCols || h.rows < 0 || h.rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (h.rows == 0) return cudaSuccess;
  Alignment l(h.cols);
  l.with(a.s.data, a.s.ld, a.s.type);
  l.with(a.dy.data, a.dy.ld, a.dy.type);
  l.with(a.ds.data, a.ds.ld, a.ds.type);
  l.with(a.dx, h.cols, a.dx_type);
  l.with(a.dresidual, h.cols, a.s.type);
  l.with(h.weight, h.cols, h.weight_type);
  return with_types(a.dx_type, a.s.type, a.dy.type, h.weight != nullptr ? h.weight_type : Elem::kF32, [&](auto types) {
    return with_run(types, l.run, [&](auto t, auto run) { return backward(a, s, t, run); });
  });
}

}  // namespace kern
}  // namespace mccl
