// Linear layer of 16-bit numbers for some tens or hundreds of rows (sm_100a): tiles of 128 x 64 or 128 x 128, a CTA each, where pairs of CTAs on tiles of
// 256 x 256 (gated.cu) would leave most of the device idle.
//
// Bound by the way to its first byte and by what each CTA loads, 128 rows of x for each 64 or 128 of W, through the second-level cache; all of it is
// in flight from the start.  A tile is done when it is: nothing overlaps what follows its product, so that is spread over the device too.
// Sums are taken out of tensor memory every 512 of the reduction and added in registers, as gated.cu does for results in 32 bits.
//
// us, bf16, launches one behind the other (B200): 64 rows of 1024 x 4096 6.5, 128 rows 6.7, 333 of 1024 x 2816 6.7, of 1000 x 2731, whose results begin
// anywhere, 10.1 (fp32 residual 10.7, gelu 11.3; pairs of CTAs 18 to 20), 1024 of 1024 x 4096, which has the larger tiles with eight warps
// each to take them out, 12.2.  About 2 of each are the launch, and 16 stages of 24 KB an SM the rest.
#include <algorithm>
#include <atomic>

#include "kernels/gated_api.h"
#include "kernels/launch_count.h"
#include "kernels/layer_epilogue.cuh"

namespace mccl {
namespace kern {
namespace {

constexpr int kRows = 128, kDepth = 64, kSms = 148;     // of a tile; k per stage
constexpr int kRowBytes = kRows * kDepth * 2;           // of x's part of a stage
constexpr int kChunk = 8;                               // stages that are added up in tensor memory
constexpr int kFirstOut = 2;
template <int kN>
constexpr int kOutWarps = kRows / 32 * (kN / kTurn);         // each has 32 rows and 64 columns
template <int kN>
constexpr int kThreads = 32 * (kFirstOut + kOutWarps<kN>);
template <int kN>
constexpr int kStageBytes = kRowBytes + kN * kDepth * 2;
template <bool kKeep, bool kWide>
constexpr int kBoxes = (kKeep ? 1 : 0) + (kWide ? 2 : 1);
template <int kN, bool kKeep, bool kWide>
constexpr int kStages = (226 * 1024 - kOutWarps<kN> * kBoxes<kKeep, kWide> * kBoxBytes) / kStageBytes<kN>;  // as many as there is room for
template <int kN, bool kKeep, bool kWide>
constexpr int kSmem = kStages<kN, kKeep, kWide> * kStageBytes<kN> + kOutWarps<kN> * kBoxes<kKeep, kWide> * kBoxBytes + 1024;

struct Tiles {
  CUtensorMap x, w, y, z, residual;
  Layer layer;
  LayerTarget target;      // without the maps
  int64_t cols;
  int tiles_i, stages;
  uint32_t x_bytes;        // of a stage
  uint32_t* failed;
  long long limit;
};

__device__ __forceinline__ uint32_t make_idesc(bool bf16, int n) {
  const uint32_t type = bf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
               "r"(static_cast<uint32_t>(accumulate))
               : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }

template <int kN, bool kKeep, bool kWide, bool kBf16>
__global__ void __launch_bounds__(kThreads<kN>, 1) layer_tiles_kernel(const __grid_constant__ Tiles w) {
  constexpr int kDepths = kStages<kN, kKeep, kWide>, kStage = kStageBytes<kN>, kOuts = kBoxes<kKeep, kWide>, kY = kKeep ? 1 : 0, kColumns = 2 * kN;
  extern __shared__ char raw[];
  __shared__ alignas(8) uint64_t bars[2 * kDepths + 5 + kOutWarps<kN>];
  __shared__ uint32_t tmem_base;
  const uint32_t smem0 = (smem_addr(raw) + 1023u) & ~1023u, bar0 = smem_addr(bars);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kDepths + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kDepths + b); };
  auto acc_free = [&](int b) { return bar0 + 8u * (2 * kDepths + 2 + b); };
  const uint32_t drained = bar0 + 8u * (2 * kDepths + 4);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kDepths; ++s) {
      bar_init(full(s), 1);
      bar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full(b), 1);
      bar_init(acc_free(b), kOutWarps<kN>);
    }
    for (int i = 0; i <= kOutWarps<kN>; ++i) bar_init(drained + 8u * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)), "n"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_base;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int ti = static_cast<int>(blockIdx.x) % w.tiles_i, tj = static_cast<int>(blockIdx.x) / w.tiles_i;
  bool ok = true, issued = false;
  if (warp == 0) {
    if (elect()) {
      int s = 0, turn = 0;
      for (int c = 0; ok && c < w.stages; ++c) {
        ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
        if (!ok) break;
        const uint32_t to = smem0 + s * kStage;
        bar_expect(full(s), w.x_bytes + kN * kDepth * 2);
        load_own_box(to + kRowBytes, &w.w, c * kDepth, tj * kN, full(s));
        load_own_box(to, &w.x, c * kDepth, ti * kRows, full(s));
        if (++s == kDepths) s = 0, ++turn;
      }
      // the products' last arrivals, before the barriers are another's
      for (int left = 0; ok && left < kDepths; ++left) {
        ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
        if (++s == kDepths) s = 0, ++turn;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect()) {
      issued = true;
      ok = w.limit > 0;  // a limit of zero, of tests: no product is issued, and all others wait in vain
      const uint32_t idesc = make_idesc(kBf16, kN);
      const uint64_t a0 = make_desc(smem0, true), b0 = make_desc(smem0 + kRowBytes, true);
      int s = 0, turn = 0, done = 0;
      for (int c = 0; ok && c < w.stages; ++done) {
        const int begin = c, end = min(w.stages, c + kChunk);
        ok = bar_wait(acc_free(done & 1), ((done >> 1) & 1) ^ 1, w.limit);
        fence_after();
        const uint32_t acc = tmem + (done & 1) * kN;
        for (; ok && c < end; ++c) {
          ok = bar_wait(full(s), turn & 1, w.limit);
          if (!ok) break;
          fence_after();
          const uint64_t a = a0 + s * (kStage >> 4), b = b0 + s * (kStage >> 4);
#pragma unroll
          for (int k = 0; k < kDepth / 16; ++k) mma(acc, a + k * step_of(true), b + k * step_of(true), idesc, c > begin || k > 0);
          mma_commit(empty(s));
          if (++s == kDepths) s = 0, ++turn;
        }
        if (ok) mma_commit(acc_full(done & 1));
      }
    }
    __syncwarp();
  } else {
    // lanes 32 q .. 32 q + 31 of tensor memory are open to the warps with warp % 4 == q
    const int q = warp & 3;
    const Layer& l = w.layer;
    const int share = (warp - kFirstOut) / 4 * kTurn;
    const int64_t col = static_cast<int64_t>(tj) * kN + share, y = static_cast<int64_t>(ti) * kRows + 32 * q, rows = w.target.rows;
    const int left = static_cast<int>(min(static_cast<int64_t>(kTurn), w.cols - col));
    const uint32_t boxes = smem0 + kDepths * kStage + (warp - kFirstOut) * (kOuts * kBoxBytes), came = drained + 8u * (1 + warp - kFirstOut);
    const bool more = l.residual != nullptr && y < rows && left > 0;
    // the residual to where y's numbers will be, while the products still run
    if (more && l.residual_vec) {
      if (lane == 0) {
        const bool two = kWide && left > 32;
        bar_expect(came, (two ? 2 : 1) * kBoxBytes);
        load_own_box(boxes + kY * kBoxBytes, &w.residual, static_cast<int>(col), static_cast<int>(y), came);
        if (two) load_own_box(boxes + (kY + 1) * kBoxBytes, &w.residual, static_cast<int>(col) + 32, static_cast<int>(y), came);
      }
    } else if (more) {
      if constexpr (kWide) {
        put_residual(l, y, rows, col, lane, boxes + kY * kBoxBytes);
      } else {
        LayerResidual r;
        r.load(l, y, rows, col, lane);
        r.put(false, lane, boxes + kY * kBoxBytes);
      }
    }
    __syncwarp();
    float v[kTurn];
#pragma unroll
    for (int i = 0; i < kTurn; ++i) v[i] = 0.f;
    int done = 0;
    for (int c = 0; c < w.stages; c += kChunk, ++done) {
      if (ok) ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_full(done & 1), (done >> 1) & 1, w.limit));
      fence_after();
      const uint32_t from = tmem + (done & 1) * kN + share + (static_cast<uint32_t>(32 * q) << 16);
#pragma unroll
      for (int i = 0; i < kTurn; i += 32) {
        float part[32];
        if (ok) {
          tmem_load<32>(from + i, part);
          tmem_wait<32>(part);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) part[e] = NAN;  // no number that looks like a result
        }
        add_to<32>(v + i, part);
      }
      fence_before();
      __syncwarp();
      if (lane == 0 && ok) bar_arrive(acc_free(done & 1));
    }
    if (left > 0) {
      const Staged<kBf16> own(boxes, lane);
      if (l.bias != nullptr)
#pragma unroll
        for (int i = 0; i < kTurn; i += 8) {
          float bias[8];
          halves<kBf16>(run_of<2>(l.bias + 2 * (col + i), w.cols - col - i, l.bias_vec), bias);
          add_to<8>(v + i, bias);
        }
      if constexpr (kKeep)
#pragma unroll
        for (int i = 0; i < kTurn; i += 8) put_z<kBf16>(own, i, v + i);
      if (l.activation != LayerActivation::kNone)
        with_activation(l.activation, [&](auto act) { Act16::values<decltype(act)::kValue, kTurn>(v); });
      if (more && l.residual_vec) ok = __all_sync(0xFFFFFFFFu, ok && bar_wait(came, 0, w.limit));
      if (!ok)
#pragma unroll
        for (int e = 0; e < kTurn; ++e) v[e] = NAN;
#pragma unroll
      for (int i = 0; i < kTurn; i += 8) {
        if (more) {
          float r[8];
          if constexpr (kWide) own.get_f32(kY, i, r);
          else halves<kBf16>(own.get(kY, i), r);
          add_to<8>(v + i, r);
        }
        if constexpr (kWide) own.put_f32(kY, i, v + i);
        else own.put(kY, i, v + i);
      }
      LayerTarget target = w.target;
      target.y_map = &w.y;
      target.z_map = &w.z;
      flush_layer<kKeep, kWide>(target, col, left, y, boxes, lane);
    }
    if (lane == 0) stores_done();
    __syncwarp();
  }
  fence_before();
  const bool failed = __syncthreads_or(!ok);
  if (failed) {
    if (threadIdx.x == 0) {
      if (w.failed) *w.failed = 1u;
      // The copies in flight, microseconds, end before this CTA's shared memory is another's.
      for (const long long begin = clock64(); clock64() - begin < kLanding;) {
      }
    }
    if (issued) {  // and the products, before tensor memory is
      mma_commit(drained);
      bar_wait(drained, 0, kWaitLimit);
    }
  }
  __syncthreads();
  fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns));
}

template <int kN, bool kKeep, bool kWide, bool kBf16>
cudaError_t run(const Tiles& w, int blocks, cudaStream_t s) {
  const auto kernel = layer_tiles_kernel<kN, kKeep, kWide, kBf16>;
  static std::atomic<uint64_t> smem_set{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (!(smem_set.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<kN, kKeep, kWide>);
    if (e != cudaSuccess) return e;
    smem_set.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads<kN>);
  cfg.dynamicSmemBytes = kSmem<kN, kKeep, kWide>;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, kernel, w);
}
template <int kN, bool kKeep, bool kWide>
cudaError_t run(const Tiles& w, bool bf16, int blocks, cudaStream_t s) {
  return bf16 ? run<kN, kKeep, kWide, true>(w, blocks, s) : run<kN, kKeep, kWide, false>(w, blocks, s);
}
template <int kN>
cudaError_t run(const Tiles& w, bool keep, bool wide, bool bf16, int blocks, cudaStream_t s) {
  if (keep) return wide ? run<kN, true, true>(w, bf16, blocks, s) : run<kN, true, false>(w, bf16, blocks, s);
  return wide ? run<kN, false, true>(w, bf16, blocks, s) : run<kN, false, false>(w, bf16, blocks, s);
}
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

int layer_tile(int64_t tokens, int64_t, int64_t out) {
  const int64_t high = ceil_div(tokens, kRows);
  return high * ceil_div(out, 64) <= kSms ? 64 : high * ceil_div(out, 128) <= kSms ? 128 : 0;
}

cudaError_t launch_layer_tiles(const LayerTiles& g, cudaStream_t s) {
  const int n = layer_tile(g.tokens, g.in, g.out);
  if (n == 0 || g.tokens <= 0 || g.in <= 0 || g.out <= 0 || encode_tiled() == nullptr) return cudaErrorInvalidValue;
  // a thread that has made no call of the runtime yet, such as autograd's, has no context, and maps need one
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e != cudaSuccess) return e;
  const LayerFinish& f = g.finish;
  Tiles w{};
  const uint32_t high = rows_read(g.tokens);
  const int64_t size = f.y_f32 ? 4 : 2, stages = ceil_div(g.in, kDepth);
  if (stages > 0x3FFFFFFF) return cudaErrorInvalidValue;
  w.target.to = g.y;
  w.target.ldo = g.out;
  w.target.rows = g.tokens;
  w.target.wide = g.out * size % 16 == 0 && reinterpret_cast<uintptr_t>(g.y) % 16 == 0;
  w.layer = layer_of(f, g.out);
  if (!make_map(&w.x, g.x, g.in, g.tokens, high, g.bf16) || !make_map(&w.w, g.weight, g.in, g.out, n, g.bf16) ||
      (w.target.wide && !make_map(&w.y, {g.y, g.out}, g.out, g.tokens, kResultRows, g.bf16, f.y_f32)) ||
      (g.z != nullptr && !make_map(&w.z, {g.z, gated_row(g.out)}, gated_row(g.out), g.tokens, kResultRows, g.bf16)) ||
      (f.residual != nullptr && w.layer.residual_vec && !make_map(&w.residual, {f.residual, f.ldr}, g.out, g.tokens, kResultRows, g.bf16, f.y_f32)))
    return cudaErrorInvalidValue;
  w.cols = g.out;
  w.tiles_i = static_cast<int>(ceil_div(g.tokens, kRows));
  w.stages = static_cast<int>(stages);
  w.x_bytes = high * kDepth * 2;
  w.failed = g.failed;
  w.limit = g.wait_limit >= 0 ? g.wait_limit : kWaitLimit;
  const int blocks = w.tiles_i * static_cast<int>(ceil_div(g.out, n));
  return n == 64 ? run<64>(w, g.z != nullptr, f.y_f32, g.bf16, blocks, s) : run<128>(w, g.z != nullptr, f.y_f32, g.bf16, blocks, s);
}

}  // namespace kern
}  // namespace mccl
