// Products of a gated feed-forward block on the fifth-generation tensor cores (sm_100a).
//
// One kernel for all six: c(i, j) = sum over k of a(i, k) b(j, k) of 16-bit numbers, added up in fp32, with what follows the
// product done on the accumulators: the activation and the product of g and u behind the first, its derivative behind the
// gradient of h.  act(z) = z s(z) with s the logistic function of z (silu) or of 2 sqrt(2/pi) (z + 0.044715 z^3) (gelu, tanh form).
//
// Rounding: h, dg and du are operands of the next product and rounded to 16 bits once.  g and u are kept for the backward pass
// with 16 significant bits (three bytes; rounded to bf16 they would put two more roundings into every gradient: 2.0 times the
// error of a result that is rounded once, where it is 1.4 so) or, where asked for, as 8-bit codes.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/gated_api.h"
#include "kernels/launch_count.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kPairs = 74;               // of SMs: a pair computes one tile
constexpr int kTile = 256;               // rows and columns of a tile; each CTA of the pair has 128 of the rows
constexpr int kHalf = 128;
constexpr int kDepth = 64;               // k per stage
constexpr int kOperand = kHalf * kDepth * 2, kStage = 2 * kOperand;   // bytes a CTA has of a stage
constexpr int kColumns = 512;            // of tensor memory: two accumulators
// warp 0 loads, warp 1 issues products, warp 2 has the tensor memory, the warps from 4 on take the accumulators out
constexpr int kLoader = 0, kIssuer = 1, kOwner = 2, kFirstOut = 4, kOutWarps = 8, kThreads = 32 * (kFirstOut + kOutWarps);

// ---- PTX ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// (What it orders is tensor memory, for which there are fences of its own: a release at cluster scope would wait for all of the
// warp's stores, a microsecond or two a tile.)
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for the phase of that parity, for four times `limit` cycles at most.  A pause of the whole device (another process has it, a
// debugger stopped it) uses up one of the four.
constexpr long long kWaitLimit = 500000000ll, kLanding = 2000000ll;  // about a quarter of a second and a millisecond
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long limit) {
  if (bar_try(bar, parity)) return true;
#pragma unroll 1
  for (int left = 4; left > 0; --left) {
    const long long begin = clock64();
    do {
      if (bar_try(bar, parity)) return true;
    } while (clock64() - begin <= limit);
  }
  return false;
}
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void store_box(const CUtensorMap* map, uint32_t from, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(from) : "memory");
}
__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All of this thread's groups have left shared memory; are done.
__device__ __forceinline__ void stores_left() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Shared-memory matrix descriptors, 128-byte swizzle.  k innermost: rows of 128 bytes (64 k), 1024 bytes per eight rows.  Own
// index innermost: rows of 128 bytes (64 of the index, one k), 1024 bytes per eight k, 8192 from 64 of the index to the next.
__device__ __forceinline__ uint64_t make_desc(uint32_t addr, bool inner) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(inner ? 1 : 8192 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// from 16 k to the next, in descriptor units
__device__ __forceinline__ uint32_t step_of(bool inner) { return (inner ? 32 : 2048) >> 4; }
__device__ __forceinline__ uint32_t make_idesc(bool bf16, bool a_inner, bool b_inner) {
  const uint32_t type = bf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (a_inner ? 0u : 1u << 15) | (b_inner ? 0u : 1u << 16) |
         (static_cast<uint32_t>(kTile >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// Arrives at this barrier of both CTAs when all products issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// kN consecutive columns of the calling thread's lane, which are there behind the wait: its operands keep whatever uses them from
// moving before it.
template <int kN>
__device__ __forceinline__ void tmem_load(uint32_t addr, float* v) {
  static_assert(kN == 16 || kN % 32 == 0, "runs of 16 or 32 columns");
  if constexpr (kN == 16) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
                   "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
                 : "r"(addr));
  } else {
#pragma unroll
    for (int i = 0; i < kN; i += 32, v += 32)
      asm volatile(
          "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
          "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
          : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
            "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]),
            "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]),
            "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
          : "r"(addr + i));
  }
}
template <int kN>
__device__ __forceinline__ void tmem_wait(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < kN; i += 16, v += 16)
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                     "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}

// ---- what a launch is told ----------------------------------------------------------------------------------
// act(z) = z s(z), s = 1 / (1 + 2^(z (c0 + c1 z^2))): silu has c0 = -log2(e) and c1 = 0, gelu 2 sqrt(2/pi) times as much and
// 0.044715 of that.  The exponent is rounded too: s is within 2^-21 + |t| 2^-22 of its size, t the logistic function's argument, the second
// only where s is small; that is 2^-15 at t = -87, where fp32 ends, and 16 bits, rounded by 2^-8 or 2^-11, do not show it.
struct Curve {
  float c0, c1;
  __device__ __forceinline__ float square(float z) const { return fminf(z * z, 1e30f); }  // no infinity for c1 = 0 to meet
  __device__ __forceinline__ float gate(float z) const {
    float e, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * fmaf(c1, square(z), c0)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    return s;
  }
  // act' = s + z s (1 - s) (c0 + 3 c1 z^2) / -log2(e)
  __device__ __forceinline__ float slope(float z, float s) const {
    return fmaf(z * (s - s * s), fmaf(-0.6931471805599453f * 3.f * c1, square(z), -0.6931471805599453f * c0), s);
  }
};

enum Out { kStore, kActivate, kDerive };  // what follows the product

struct Finish {
  bool bf16;
  Curve curve;
  char* kept;
  int64_t rows, pitch;    // of what is kept, and of h, dg and du
};
// One product: tiles, and how they become items of work.
struct Job {
  CUtensorMap a[2], b[2], out[3];
  void* to[3];
  int64_t rows, cols, ldo;  // of one result; cols: of h, dg and du their pitch
  bool a_inner, b_inner;    // k innermost
  uint32_t bytes;           // of a stage, that both CTAs load
  bool wide;                // there are maps of the results: their rows are aligned to 16 bytes
  int rows_segment;         // tiles of rows of the first of two results (dWg, then dWu); all of them where there is one
  int tiles_i, tiles_j;     // tiles_i: of all results
  int stages, segment;      // of the reduction; stages of its first part (dg Wg, then du Wu)
  int first;                // item
  int whole;                // items that are whole tiles; behind them tiles whose reduction `splits` pairs share, with partial sums from `part` on
  int splits, per_split, part;
  int join;                 // the first such tile among those of all jobs
};
constexpr int kMostJobs = 3;
template <Out kOut>
constexpr int kJobs = kOut == kStore ? kMostJobs : 1;
template <int kN>
struct Work {
  Job job[kN];
  Finish f;
  int jobs, items;
  float* partial;
  uint32_t* failed;
  long long limit;
};

// A tile's place, so that the pairs at work at a time read few rows of each operand: kBand tiles of rows, column by column.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_place(const Job& j, int tile, int& ti, int& tj) {
  const int band = tile / (kBand * j.tiles_j), in_band = tile - band * kBand * j.tiles_j;
  const int high = min(kBand, j.tiles_i - band * kBand);
  tj = in_band / high;
  ti = band * kBand + in_band - tj * high;
}
struct Item {
  int job, ti, tj, c0, c1, part;  // part: which partial sum, or -1
  template <int kN>
  __device__ __forceinline__ Item(const Work<kN>& w, int item) {
    job = 0;
    while (job + 1 < w.jobs && item >= w.job[job + 1].first) ++job;
    const Job& j = w.job[job];
    item -= j.first;
    if (item < j.whole) {
      tile_place(j, item, ti, tj);
      c0 = 0;
      c1 = j.stages;
      part = -1;
    } else {
      part = item - j.whole;
      const int t = part / j.splits;
      tile_place(j, j.whole + t, ti, tj);
      c0 = (part - t * j.splits) * j.per_split;
      c1 = min(j.stages, c0 + j.per_split);
      part += j.part;
    }
  }
};
// A pair's items.  Several jobs come the longest items first: the pair that had the longest of the first round gets the shortest of the
// others.
__device__ __forceinline__ int item_of(int round, int pair, int pairs, int jobs) {
  return round * pairs + (round > 0 && jobs > 1 ? pairs - 1 - pair : pair);
}

// ---- after the product --------------------------------------------------------------------------------------
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kBf16) return store_pair<__nv_bfloat16>(a, b);
  else return store_pair<__half>(a, b);
}

// Floats of three bytes: the upper 24 bits, rounded to nearest; infinities and NaN cut off.
__device__ __forceinline__ uint32_t three_bytes(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x7F800000u) == 0x7F800000u ? b | (b & 0x7FFFFFu ? 0x400000u : 0u) : b + 0x80u;
}

// Where g and u wait: blocks of 8 (three bytes: 16 of upper, 8 of lower ones) or 16 columns (codes) of all tokens, one behind the
// other, so that neighbouring rows, which neighbouring lanes have, lie side by side.
struct Wide {
  uint4* upper[2];
  uint2* lower[2];
  __device__ __forceinline__ Wide(char* kept, int64_t rows, int64_t pitch) {
    const int64_t n = rows * pitch;
    upper[0] = reinterpret_cast<uint4*>(kept);
    upper[1] = reinterpret_cast<uint4*>(kept + 2 * n);
    lower[0] = reinterpret_cast<uint2*>(kept + 4 * n);
    lower[1] = reinterpret_cast<uint2*>(kept + 5 * n);
  }
};
struct Eight {
  uint4* codes[2];
  float* scales[2];
  __device__ __forceinline__ Eight(char* kept, int64_t rows, int64_t pitch) {
    const int64_t n = rows * pitch;
    codes[0] = reinterpret_cast<uint4*>(kept);
    codes[1] = reinterpret_cast<uint4*>(kept + n);
    scales[0] = reinterpret_cast<float*>(kept + 2 * n);
    scales[1] = scales[0] + rows * (pitch / kGroup8);
  }
};
__device__ __forceinline__ void keep_wide(const Wide& k, int which, int64_t at, const float* v) {  // 8 numbers
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = three_bytes(v[i]);
  __stcs(k.upper[which] + at, make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632), __byte_perm(b[4], b[5], 0x7632),
                                         __byte_perm(b[6], b[7], 0x7632)));
  __stcs(k.lower[which] + at, make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0051), __byte_perm(b[2], b[3], 0x0051), 0x5410),
                                  __byte_perm(__byte_perm(b[4], b[5], 0x0051), __byte_perm(b[6], b[7], 0x0051), 0x5410)));
}
__device__ __forceinline__ void take_wide(const uint4& up, const uint2& low, float* v) {
  const uint32_t u[4] = {up.x, up.y, up.z, up.w}, l[2] = {low.x, low.y};
#pragma unroll
  for (int i = 0; i < 8; ++i)  // the two upper bytes, the lower one, and nothing
    v[i] = __uint_as_float(__byte_perm(u[i / 2], l[i / 4], (i % 2 ? 0x3200 : 0x1000) | (4 + i % 4) << 4) & 0xFFFFFF00u);
}

// Where 8 numbers of a thread's row go, `i` columns from where it is: straight to memory, which costs a request for each row (the
// joining kernel), or to the warp's boxes of 32 rows and 64 columns in shared memory, 128-byte swizzle,
// which then leave as a whole.  (Straight to memory kGate took 99 us of 8192 x 1024 x 2816, bound by its requests.)
constexpr int kTurn = 64, kBoxBytes = 32 * kTurn * 2;
template <bool kBf16>
struct Direct {
  uint16_t* out[3];
  int64_t left;  // numbers of the row from here on, a multiple of 8
  __device__ __forceinline__ void put(int which, int i, const float* v) const {
    if (i < left)
      *reinterpret_cast<uint4*>(out[which] + i) =
          make_uint4(pack2<kBf16>(v[0], v[1]), pack2<kBf16>(v[2], v[3]), pack2<kBf16>(v[4], v[5]), pack2<kBf16>(v[6], v[7]));
  }
};
template <bool kBf16>
struct Staged {
  uint32_t row;       // of the first box
  int swizzle;
  __device__ __forceinline__ Staged(uint32_t boxes, int lane) : row(boxes + lane * 128), swizzle(lane & 7) {}
  __device__ __forceinline__ void put(int which, int i, const float* v) const {
    const uint32_t to = row + which * kBoxBytes + ((i / 8) ^ swizzle) * 16;
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(pack2<kBf16>(v[0], v[1])), "r"(pack2<kBf16>(v[2], v[3])),
                 "r"(pack2<kBf16>(v[4], v[5])), "r"(pack2<kBf16>(v[6], v[7]))
                 : "memory");
  }
};
// kN columns of g and u to h and to what is kept.
template <GatedKeep kKeep, int kN, typename Sink>
__device__ __forceinline__ void finish_activate(const Finish& f, int64_t row, int64_t col, const float* g, const float* u, const Sink& sink, int i0) {
  const bool there = row < f.rows;
  if (kKeep == GatedKeep::kEight && there) {
    static_assert(kKeep != GatedKeep::kEight || kN == kGroup8, "a thread has a whole group");
    const Eight k(f.kept, f.rows, f.pitch);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float* v = which ? u : g;
      uint32_t most = 0u;
#pragma unroll
      for (int i = 0; i < kN; ++i) most = most8(most, v[i]);
      const Scale8 s = scale8(__uint_as_float(most));
      k.scales[which][col / kGroup8 * f.rows + row] = s.scale;
#pragma unroll
      for (int i = 0; i < kN; i += 16)
        k.codes[which][(col + i) / 16 * f.rows + row] =
            make_uint4(codes8(v[i], v[i + 1], v[i + 2], v[i + 3], s.inverse), codes8(v[i + 4], v[i + 5], v[i + 6], v[i + 7], s.inverse),
                       codes8(v[i + 8], v[i + 9], v[i + 10], v[i + 11], s.inverse), codes8(v[i + 12], v[i + 13], v[i + 14], v[i + 15], s.inverse));
    }
  }
#pragma unroll
  for (int i = 0; i < kN; i += 8) {
    if (kKeep == GatedKeep::kWide && there) {
      const Wide k(f.kept, f.rows, f.pitch);
      const int64_t at = (col + i) / 8 * f.rows + row;
      keep_wide(k, 0, at, g + i);
      keep_wide(k, 1, at, u + i);
    }
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = g[i + e] * f.curve.gate(g[i + e]) * u[i + e];
    sink.put(0, i0 + i, h);
  }
}
// 16 columns of g and u as they were kept.
template <GatedKeep kKeep>
struct Kept {
  uint4 upper[2][2];
  uint2 lower[2][2];
  __device__ __forceinline__ void load(const Finish& f, int64_t row, int64_t col) {
    const Wide k(f.kept, f.rows, f.pitch);
    const int64_t at = col / 8 * f.rows + row;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        upper[which][b] = __ldcs(k.upper[which] + at + b * f.rows);
        lower[which][b] = __ldcs(k.lower[which] + at + b * f.rows);
      }
  }
  __device__ __forceinline__ void value(int b, float* g, float* u) const {  // 8 of them
    take_wide(upper[0][b], lower[0][b], g);
    take_wide(upper[1][b], lower[1][b], u);
  }
};
template <>
struct Kept<GatedKeep::kEight> {
  uint4 codes[2];
  float scale[2];
  __device__ __forceinline__ void load(const Finish& f, int64_t row, int64_t col) {
    const Eight k(f.kept, f.rows, f.pitch);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      codes[which] = __ldcs(k.codes[which] + col / 16 * f.rows + row);
      scale[which] = __ldg(k.scales[which] + col / kGroup8 * f.rows + row);
    }
  }
  __device__ __forceinline__ void value(int b, float* g, float* u) const {
    values8(b ? codes[0].z : codes[0].x, scale[0], g);
    values8(b ? codes[0].w : codes[0].y, scale[0], g + 4);
    values8(b ? codes[1].z : codes[1].x, scale[1], u);
    values8(b ? codes[1].w : codes[1].y, scale[1], u + 4);
  }
};
// 16 columns of dh to h, dg and du.
template <GatedKeep kKeep, typename Sink>
__device__ __forceinline__ void finish_derive(const Finish& f, const float* dh, const Kept<kKeep>& kept, const Sink& sink, int i0) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    float g[8], u[8], h[8], dg[8], du[8];
    kept.value(b, g, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = dh[8 * b + e], s = f.curve.gate(g[e]), a = g[e] * s;
      h[e] = a * u[e];
      du[e] = d * a;
      dg[e] = d * u[e] * f.curve.slope(g[e], s);
    }
    sink.put(0, i0 + 8 * b, h);
    sink.put(1, i0 + 8 * b, dg);
    sink.put(2, i0 + 8 * b, du);
  }
}

// ---- product ------------------------------------------------------------------------------------------------
// The columns that a thread takes out of the accumulator at a time (of h for kActivate: of c two each; an 8-bit group is one
// thread's).  64 columns leave together.
template <Out kOut, GatedKeep kKeep>
constexpr int kTake = kOut == kActivate && kKeep == GatedKeep::kEight ? 64 : 16;
template <Out kOut>
constexpr int kBoxes = kOut == kDerive ? 3 : 1;
template <Out kOut>
constexpr int kStages = kOut == kDerive ? 4 : 6;
template <Out kOut>
constexpr int kSmem = kStages<kOut> * kStage + kOutWarps * kBoxes<kOut> * kBoxBytes + 1024;  // of 227 KB

constexpr int kJoinThreads = 256;
template <Out kOut, GatedKeep kKeep>
constexpr int kJoinSmem = kTake<kOut, kKeep> * (kOut == kActivate ? 2 : 1) * kHalf * 4;

// What a thread needs from memory for its first columns of a tile is asked for while the products still run, for the next ones while
// it is busy with these.
struct Nothing {
  __device__ __forceinline__ void load(const Finish&, int64_t, int64_t) {}
};
template <Out kOut, GatedKeep kKeep>
using Ahead = std::conditional_t<kOut == kDerive, Kept<kKeep>, Nothing>;

// A thread's row and columns of a tile: `row` of the result that the tile is of, its columns from `col` on.
struct Spot {
  int64_t row, col;
  int which;      // kStore: which of two results
};
template <Out kOut>
__device__ __forceinline__ Spot spot_of(const Job& j, int ti, int tj, int row_in_tile) {
  const int second = kOut == kStore && ti >= j.rows_segment;
  return {static_cast<int64_t>(second ? ti - j.rows_segment : ti) * kTile + row_in_tile, static_cast<int64_t>(tj) * (kOut == kActivate ? kHalf : kTile), second};
}
// kCols columns from `c` of the tile on, into a sink.
template <Out kOut, GatedKeep kKeep, int kCols, typename Fetch, typename Sink>
__device__ __forceinline__ void finish_turn(const Finish& f, const Spot& at, int c, int last, Ahead<kOut, kKeep>& ahead, const Fetch& fetch, const Sink& sink) {
  constexpr int kN = kTake<kOut, kKeep>;
#pragma unroll 1
  for (int i = 0; i < kCols; i += kN) {
    if constexpr (kOut == kActivate) {
      float g[kN], u[kN];
      fetch(c + i, g);
      fetch(kHalf + c + i, u);
      finish_activate<kKeep, kN>(f, at.row, at.col + c + i, g, u, sink, i);
    } else {
      float v[kN];
      if constexpr (kOut == kDerive) {
        const Kept<kKeep> now = ahead;
        if (c + i + kN < last) ahead.load(f, min(at.row, f.rows - 1), at.col + c + i + kN);
        fetch(c + i, v);
        finish_derive<kKeep>(f, v, now, sink, i);
      } else {
        fetch(c + i, v);
#pragma unroll
        for (int e = 0; e < kN; e += 8) sink.put(0, i + e, v + e);
      }
    }
  }
}
// A pair of CTAs per tile of 256 x 256, tiles in turn: each CTA loads half of either operand's rows and has half of the
// accumulator's; the first one issues the products of both.  Two accumulators, so that a tile is taken out while the next one
// is multiplied.  A stage is 64 KB for 8.4 million multiplications: what passes through the second-level cache, 13.5 TB/s of it, bounds
// all of them.  8192 x 1024 x 2816 bf16 (B200, by itself): up 61 us without, 79 with three kept bytes, 71 with codes (1.55, 1.20, 1.33
// PFLOP/s), down 34 (1.39), gate 75 and 67 (0.63 and 0.71: 12 or 8 bytes a number of its own beside the operands, 10.8 TB/s), the last three 168
// (1.40); 16384 x 2048 x 5632 up 545 (1.39), down 240 (1.58), gate 366, the last three 1250 (1.51).
// Left: 16 warps to take the accumulators out (no faster, 397 for 339 of the wide gate), what was kept asked for two runs ahead through
// shared memory (72 for 75, but 418 for 379 of the wide one, which has then a stage less) or a tile ahead into the second-level cache
// (83 and 431).
template <Out kOut, GatedKeep kKeep>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gated_kernel(const __grid_constant__ Work<kJobs<kOut>> w) {
  constexpr int kDepths = kStages<kOut>, kOuts = kBoxes<kOut>;
  extern __shared__ char raw[];
  __shared__ alignas(8) uint64_t bars[2 * kDepths + 5];
  __shared__ uint32_t tmem_base;
  const uint32_t smem0 = (smem_addr(raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t bar0 = smem_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kDepths + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kDepths + b); };
  auto acc_free = [&](int b) { return bar0 + 8u * (2 * kDepths + 2 + b); };
  const uint32_t drained = bar0 + 8u * (2 * kDepths + 4);
  if (tid == 0) {
    for (int s = 0; s < kDepths; ++s) {
      bar_init(full(s), 1);
      bar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      bar_init(acc_full(b), 1);
      bar_init(acc_free(b), 2 * kOutWarps);
    }
    bar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kOwner) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)), "n"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  __syncwarp();
  fence_before();
  cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_base;
  // Only now, when all that came before is done: copies beside this (gated_copies_kernel) do not wait before they write.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  bool ok = true, issued = false;

  if (warp == kLoader) {
    if (elect()) {
      int s = 0, turn = 0;
      for (int round = 0, item = pair; ok && item < w.items; item = item_of(++round, pair, pairs, w.jobs)) {
        const Item t(w, item);
        const Job& j = w.job[t.job];
        const int i_second = t.ti >= j.rows_segment, i0 = (i_second ? t.ti - j.rows_segment : t.ti) * kTile + rank * kHalf;
        // g and u side by side: one CTA has the rows of Wg, the other those of Wu
        const int j0 = kOut == kActivate ? t.tj * kHalf : t.tj * kTile + rank * kHalf;
        const bool a_inner = j.a_inner, b_inner = j.b_inner;
        for (int c = t.c0; ok && c < t.c1; ++c) {
          ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
          if (!ok) break;
          const int k_second = c >= j.segment, k0 = (k_second ? c - j.segment : c) * kDepth;
          const CUtensorMap* a = &j.a[i_second | k_second];
          const CUtensorMap* b = &j.b[kOut == kActivate ? rank : k_second];
          const uint32_t to = smem0 + s * kStage, bar = in_leader(full(s));
          if (rank == 0) bar_expect(full(s), j.bytes);
          if (a_inner) load_box(to, a, k0, i0, bar);
          else {
            load_box(to, a, i0, k0, bar);
            load_box(to + kOperand / 2, a, i0 + 64, k0, bar);
          }
          if (b_inner) load_box(to + kOperand, b, k0, j0, bar);
          else {
            load_box(to + kOperand, b, j0, k0, bar);
            load_box(to + kOperand + kOperand / 2, b, j0 + 64, k0, bar);
          }
          if (++s == kDepths) s = 0, ++turn;
        }
      }
      // the products' last arrivals, before the barriers are another's
      for (int left = 0; ok && left < kDepths; ++left) {
        ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
        if (++s == kDepths) s = 0, ++turn;
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    if (rank == 0 && elect()) {
      issued = true;
      ok = w.limit > 0;  // a limit of zero, of tests: no product is issued, and all others wait in vain
      int s = 0, turn = 0, done = 0;
      for (int round = 0, item = pair; ok && item < w.items; item = item_of(++round, pair, pairs, w.jobs), ++done) {
        const Item t(w, item);
        const bool a_inner = w.job[t.job].a_inner, b_inner = w.job[t.job].b_inner;
        const uint32_t idesc = make_idesc(w.f.bf16, a_inner, b_inner), step_a = step_of(a_inner), step_b = step_of(b_inner);
        const uint64_t a0 = make_desc(smem0, a_inner), b0 = make_desc(smem0 + kOperand, b_inner);
        const int buffer = done & 1;
        ok = bar_wait(acc_free(buffer), ((done >> 1) & 1) ^ 1, w.limit);
        fence_after();
        const uint32_t acc = tmem + buffer * kTile;
        for (int c = t.c0; ok && c < t.c1; ++c) {
          ok = bar_wait(full(s), turn & 1, w.limit);
          if (!ok) break;
          fence_after();
          const uint64_t a = a0 + s * (kStage >> 4), b = b0 + s * (kStage >> 4);
#pragma unroll
          for (int k = 0; k < kDepth / 16; ++k) mma(acc, a + k * step_a, b + k * step_b, idesc, c > t.c0 || k > 0);
          mma_commit(empty(s));
          if (++s == kDepths) s = 0, ++turn;
        }
        if (ok) mma_commit(acc_full(buffer));
      }
    }
    __syncwarp();
  } else if (warp >= kFirstOut) {
    // lanes 32 q .. 32 q + 31 of tensor memory are open to the warps with warp % 4 == q, which share the columns
    constexpr int kN = kTake<kOut, kKeep>, kShares = kOutWarps / 4, kShare = (kOut == kActivate ? kHalf : kTile) / kShares;
    const int q = warp & 3, share = (warp - kFirstOut) >> 2;
    const int row = rank * kHalf + 32 * q + lane;
    const uint32_t boxes = smem0 + kDepths * kStage + (warp - kFirstOut) * (kOuts * kBoxBytes);
    int done = 0;
    for (int round = 0, item = pair; item < w.items; item = item_of(++round, pair, pairs, w.jobs), ++done) {
      const Item t(w, item);
      const Job& j = w.job[t.job];
      const int buffer = done & 1;
      const Spot at = spot_of<kOut>(j, t.ti, t.tj, row);
      Ahead<kOut, kKeep> ahead;
      if (t.part < 0 && at.col + share * kShare < j.cols) ahead.load(w.f, min(at.row, w.f.rows - 1), at.col + share * kShare);
      if (ok) ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_full(buffer), (done >> 1) & 1, w.limit));
      fence_after();
      const uint32_t from = tmem + buffer * kTile + (static_cast<uint32_t>(32 * q) << 16);
      auto fetch = [&](int c, float* v) {
        if (ok) {
          tmem_load<kN>(from + c, v);
          tmem_wait<kN>(v);
        } else {
#pragma unroll
          for (int i = 0; i < kN; ++i) v[i] = NAN;  // no number that looks like a result
        }
      };
      if (t.part < 0) {
        const int64_t left = j.cols - at.col;
        const int first = share * kShare, last = static_cast<int>(min(static_cast<int64_t>(first + kShare), left));
        const int64_t y = at.row - lane;  // the warp's first row
#pragma unroll 1
        for (int c = first; c < last; c += kTurn) {
          if (lane == 0) stores_left();
          __syncwarp();
          if (w.f.bf16) finish_turn<kOut, kKeep, kTurn>(w.f, at, c, last, ahead, fetch, Staged<true>(boxes, lane));
          else finish_turn<kOut, kKeep, kTurn>(w.f, at, c, last, ahead, fetch, Staged<false>(boxes, lane));
          if (kOut != kStore || j.wide) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (y < j.rows)
#pragma unroll
                for (int b = 0; b < kOuts; ++b)
                  store_box(&j.out[kOut == kDerive ? b : at.which], boxes + b * kBoxBytes, static_cast<int>(at.col) + c, static_cast<int>(y));
              stores_commit();
            }
          } else {  // rows that are not aligned: two numbers a lane, row by row
            __syncwarp();
            const int n = static_cast<int>(min(static_cast<int64_t>(32), j.rows - y));
            uint16_t* to = static_cast<uint16_t*>(j.to[at.which]) + y * j.ldo + at.col + c + 2 * lane;
            const int here = last - c - 2 * lane;
#pragma unroll 4
            for (int r = 0; r < n; ++r, to += j.ldo) {
              uint32_t v;
              asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(boxes + r * 128 + (((lane / 4) ^ (r & 7)) * 16) + lane % 4 * 4));
              if (here > 0) to[0] = static_cast<uint16_t>(v);
              if (here > 1) to[1] = static_cast<uint16_t>(v >> 16);
            }
            __syncwarp();
          }
        }
      } else {
        float* to = w.partial + static_cast<int64_t>(t.part) * (kTile * kTile) + row;
#pragma unroll 1
        for (int c = share * (kTile / kShares); c < (share + 1) * (kTile / kShares); c += kN) {
          float v[kN];
          fetch(c, v);
          if (at.row < j.rows)
#pragma unroll
            for (int i = 0; i < kN; ++i) __stcg(to + static_cast<int64_t>(c + i) * kTile, v[i]);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0 && ok) bar_arrive_cluster(in_leader(acc_free(buffer)));
    }
    if (lane == 0) stores_done();
    __syncwarp();
  }
  fence_before();
  const bool failed = __syncthreads_or(!ok);
  if (failed) {
    if (tid == 0) {
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
  cluster_sync();
  fence_after();
  if (warp == kOwner) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns));
}

// Adds up the parts of the tiles whose reduction was shared, in order, and finishes them.  A block has 16 (64) columns of half a
// tile: its warps add up two columns each, four rows a lane, and hand them over in shared memory to the thread that has the row.
// (Each thread its own row's numbers: 14.5 us for 18 MB of parts, a quarter of it in flight.)
template <Out kOut, GatedKeep kKeep>
__global__ void __launch_bounds__(kJoinThreads) gated_join_kernel(const __grid_constant__ Work<kJobs<kOut>> w) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kN = kTake<kOut, kKeep>, kAll = kN * (kOut == kActivate ? 2 : 1), kWarps = kJoinThreads / 32, kEach = kAll / kWarps, kAt = 2, kParts = 8;
  extern __shared__ float4 sums[];  // [kAll][32]
  int job = 0;
  while (job + 1 < w.jobs && static_cast<int>(blockIdx.x) >= w.job[job + 1].join) ++job;
  const Job& j = w.job[job];
  const int tile = static_cast<int>(blockIdx.x) - j.join, c = blockIdx.z * kN, row = blockIdx.y * kHalf + threadIdx.x % kHalf, lane = threadIdx.x % 32,
            warp = threadIdx.x / 32;
  int ti, tj;
  tile_place(j, j.whole + tile, ti, tj);
  const Finish& f = w.f;
  const Spot at = spot_of<kOut>(j, ti, tj, row);
  const int64_t left = j.cols - at.col - c;
  if (left <= 0 || at.row - threadIdx.x % kHalf >= j.rows) return;
  const float* from = w.partial + (j.part + static_cast<int64_t>(tile) * j.splits) * (kTile * kTile) + blockIdx.y * kHalf + 4 * lane;
#pragma unroll 1
  for (int i0 = 0; i0 < kEach; i0 += kAt) {
    float4 sum[kAt];
    const float* column[kAt];
#pragma unroll
    for (int i = 0; i < kAt; ++i) {
      const int col = warp + kWarps * (i0 + i);
      column[i] = from + (col < kN ? c + col : kHalf + c + col - kN) * kTile;
      sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int p = 0; p < j.splits; p += kParts) {
      float4 x[kAt][kParts];
#pragma unroll
      for (int q = 0; q < kParts; ++q)
#pragma unroll
        for (int i = 0; i < kAt; ++i)
          if (p + q < j.splits) x[i][q] = __ldcg(reinterpret_cast<const float4*>(column[i] + static_cast<int64_t>(p + q) * (kTile * kTile)));
#pragma unroll
      for (int q = 0; q < kParts; ++q)
#pragma unroll
        for (int i = 0; i < kAt; ++i)
          if (p + q < j.splits) {
            sum[i].x += x[i][q].x;
            sum[i].y += x[i][q].y;
            sum[i].z += x[i][q].z;
            sum[i].w += x[i][q].w;
          }
    }
#pragma unroll
    for (int i = 0; i < kAt; ++i) sums[(warp + kWarps * (i0 + i)) * 32 + lane] = sum[i];
  }
  __syncthreads();
  const int mine = threadIdx.x % kHalf;  // the second half of the threads has no row
  auto fetch = [&](int col, float* v) {
    const float* s = reinterpret_cast<const float*>(sums) + (col >= kHalf && kOut == kActivate ? kN : 0) * kHalf + mine;
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = s[i * kHalf];
  };
  if constexpr (kOut == kStore) {
    if (!j.wide) {  // rows that are not aligned: handed over once more, two of them a warp and turn
      float v[kN];
      fetch(c, v);
      __syncthreads();
      uint32_t* rows = reinterpret_cast<uint32_t*>(sums);  // [128][9]
#pragma unroll
      for (int i = 0; i < kN; i += 2)
        if (threadIdx.x < kHalf) rows[mine * 9 + i / 2] = f.bf16 ? pack2<true>(v[i], v[i + 1]) : pack2<false>(v[i], v[i + 1]);
      __syncthreads();
      const int64_t y = at.row - mine;
      uint16_t* to = static_cast<uint16_t*>(j.to[at.which]) + at.col + c;
      for (int i = threadIdx.x; i < kHalf * kN; i += kJoinThreads) {
        const int r = i / kN, e = i % kN;
        if (y + r < j.rows && e < left) to[(y + r) * j.ldo + e] = static_cast<uint16_t>(rows[r * 9 + e / 2] >> (16 * (e % 2)));
      }
      return;
    }
  }
  if (threadIdx.x >= kHalf || at.row >= j.rows) return;
  Ahead<kOut, kKeep> ahead;
  ahead.load(f, at.row, at.col + c);
  const int64_t to = at.row * j.ldo + at.col + c;
  uint16_t* const out[3] = {static_cast<uint16_t*>(j.to[at.which]) + to, static_cast<uint16_t*>(j.to[1]) + to, static_cast<uint16_t*>(j.to[2]) + to};
  if (f.bf16) finish_turn<kOut, kKeep, kN>(f, at, c, c + kN, ahead, fetch, Direct<true>{{out[0], out[1], out[2]}, left});
  else finish_turn<kOut, kKeep, kN>(f, at, c, c + kN, ahead, fetch, Direct<false>{{out[0], out[1], out[2]}, left});
}

// ---- rows that are not aligned --------------------------------------------------------------------------------
struct Copies {
  GatedCopy job[kGatedCopies];
  int64_t first[kGatedCopies + 1];  // blocks
};
constexpr int kCopyRows = 8, kCopyCols = 512;  // of a block; a warp has a row, two neighbours a lane and turn
constexpr int kCopyThreads = 32 * kCopyRows;
// Ahead of the product that reads them, or beside the product before it.  (333 tokens of 1000 x 2731, w_down copied, 35 us ahead of
// both products, 27 beside the first.)
__global__ void __launch_bounds__(kCopyThreads) gated_copies_kernel(const Copies w) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int j = 0;
  while (static_cast<int64_t>(blockIdx.x) >= w.first[j + 1]) ++j;
  const GatedCopy& c = w.job[j];
  const int64_t across = (c.cols + kCopyCols - 1) / kCopyCols, block = blockIdx.x - w.first[j];
  const int64_t row = block / across * kCopyRows + threadIdx.x / 32, col = block % across * kCopyCols + threadIdx.x % 32 * 2;
  // What waits for this grid waits for the product beside it too: one thread's wait is enough, the first one's, which has a row.
  if (row >= c.rows) return;
  const uint16_t* from = static_cast<const uint16_t*>(c.from) + row * c.row_stride;
  uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(c.to) + row * c.ld);
  uint32_t v[kCopyCols / 64];
#pragma unroll
  for (int i = 0; i < kCopyCols / 64; ++i) {
    const int64_t at = col + 64 * i;
    v[i] = (at < c.cols ? from[at * c.col_stride] : 0u) | (at + 1 < c.cols ? static_cast<uint32_t>(from[(at + 1) * c.col_stride]) << 16 : 0u);
  }
#pragma unroll
  for (int i = 0; i < kCopyCols / 64; ++i)
    if (col + 64 * i < c.cols) to[(col + 64 * i) / 2] = v[i];
  if (blockIdx.x == 0 && threadIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- host ---------------------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Sizes {
  int64_t rows, cols, depth;   // of one result, and of one part of the reduction
  int results, parts;          // results beside each other in the rows; parts of the reduction
  bool gate;                   // a tile has 128 columns of two results
};
Sizes sizes_of(GatedProduct p, const GatedShape& s) {
  switch (p) {
    case GatedProduct::kUp: return {s.tokens, s.hidden, s.width, 1, 1, true};
    case GatedProduct::kDown: return {s.tokens, s.width, s.hidden, 1, 1, false};
    case GatedProduct::kGate: return {s.tokens, s.hidden, s.width, 1, 1, false};
    case GatedProduct::kInput: return {s.tokens, s.width, s.hidden, 1, 2, false};
    case GatedProduct::kWeightUp: return {s.hidden, s.width, s.tokens, 2, 1, false};
    default: return {s.width, s.hidden, s.tokens, 1, 1, false};
  }
}
struct Plan {
  int64_t tiles_i, tiles_j, stages, segment;
  int64_t whole, tail, splits, per_split;   // tail: tiles that are shared along the reduction
  int64_t longest() const { return whole > 0 ? stages : per_split; }
};
constexpr double kStageUs = 0.37;
// Whether sharing tiles along the reduction saves more than it costs: a partial sum is written and read at 6 TB/s, behind 2 us for
// the launch that adds them up.  us, shared and not: down of 1024 tokens of 1024 x 2816 15.4 and 18.9, of 1000 of 768 x 2048 13.9 and 15.5;
// up of 2048 tokens of 2048 x 4096 (which stays whole) 51.3 and 46.8.
bool split_pays(const Plan& l, int64_t tiles, int64_t splits, int64_t per, int64_t rows) {
  const double saved = kStageUs * static_cast<double>(l.stages - per);
  return saved > 2.0 + 8.0 * static_cast<double>(tiles * splits * kTile * std::min<int64_t>(kTile, rows)) / 6e6;
}
Plan plan_of(GatedProduct p, const GatedShape& s) {
  const Sizes z = sizes_of(p, s);
  Plan l{};
  l.tiles_i = ceil_div(z.rows, kTile) * z.results;
  l.tiles_j = ceil_div(z.cols, z.gate ? kHalf : kTile);
  l.segment = ceil_div(z.depth, kDepth);
  l.stages = l.segment * z.parts;
  l.whole = l.tiles_i * l.tiles_j;
  l.splits = 1;
  l.per_split = l.stages;
  return l;
}
void share(Plan& l, int64_t tiles, int64_t most, int64_t rows) {
  most = std::min<int64_t>({most, l.stages / 4, 16});
  if (most < 2) return;
  const int64_t per = ceil_div(l.stages, most), splits = ceil_div(l.stages, per);
  if (!split_pays(l, tiles, splits, per, rows)) return;
  l.whole -= tiles;
  l.tail = tiles;
  l.splits = splits;
  l.per_split = per;
}
// One product: whole tiles as long as they fill the device; the rest, less than one tile a pair, is shared along the reduction where that
// pays.
void plan_one(GatedProduct p, const GatedShape& s, Plan& l) {
  l = plan_of(p, s);
  const int64_t tail = l.whole % kPairs;
  if (tail > 0) share(l, tail, kPairs / tail, sizes_of(p, s).rows);
}
// Stages that a product by itself takes, with 8 us for sums that are joined and 4 for a launch.
double stages_alone(const Plan& l) {
  const int64_t rounds = ceil_div(l.whole, kPairs);
  return static_cast<double>(rounds * l.stages + (l.tail > 0 ? l.per_split : 0)) + (l.tail > 0 ? 12.0 : 4.0) / kStageUs;
}
// Several products side by side: whole tiles, but for a product whose tiles are so few and long that the device would wait for them.
// Whether that is faster than one after the other, of which each leaves part of the device idle in its last round: 8192 tokens of 1024 x
// 2816 168 us and 183, 1024 32 and 47, 64 of 640 x 2112 13 and 25; 16384 of 2048 x 5632, fourteen rounds, 1302 and 1246, for what
// different operands in the second-level cache cost (a twentieth, taken into account).
bool plan_together(const GatedProduct* p, const GatedShape& s, int n, Plan* l, int* order) {
  int64_t total = 0;
  double alone = 0;
  for (int i = 0; i < n; ++i) {
    Plan one{};
    plan_one(p[i], s, one);
    alone += stages_alone(one);
    l[i] = plan_of(p[i], s);
    total += l[i].whole * l[i].stages;
    order[i] = i;
  }
  const int64_t fair = std::max<int64_t>(ceil_div(total, kPairs), 8);
  bool joins = false;
  for (int i = 0; i < n; ++i) {
    if (2 * l[i].stages > 3 * fair) share(l[i], l[i].whole, ceil_div(l[i].stages, fair), sizes_of(p[i], s).rows);
    joins = joins || l[i].tail > 0;
  }
  std::sort(order, order + n, [&](int a, int b) { return l[a].longest() != l[b].longest() ? l[a].longest() > l[b].longest() : a < b; });
  int64_t tiles = 0;
  for (int i = 0; i < n; ++i) tiles += l[i].whole;
  if (tiles > 40 * kPairs) return false;  // little idle in so many rounds, and long to add up
  // what the pair with the most to do has: item_of's order
  int64_t load[kPairs] = {}, most = 0, item = 0;
  for (int i = 0; i < n; ++i) {
    const Plan& q = l[order[i]];
    for (int64_t t = 0; t < q.whole + q.tail * q.splits; ++t, ++item) {
      const int64_t round = item / kPairs, at = item % kPairs;
      int64_t& mine = load[round > 0 ? kPairs - 1 - at : at];
      mine += q.longest();
      most = std::max(most, mine);
    }
  }
  return 1.05 * static_cast<double>(most) + (joins ? 12.0 : 4.0) / kStageUs < alone;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}
// A matrix of `outer` rows of `inner` numbers in boxes of 64 of a row and of `box_rows` rows: read, of 128 (k innermost; of tokens fewer
// where there are fewer: a box's rows beyond the matrix take time, 73 us for 67 of 12 tokens of 4096 x 10240, 279 for 236 of 3 of 8192 x
// 24576; what lies below in shared memory are rows of nobody's) or 64 (own index innermost); written, of 32.
constexpr uint32_t kOwnRows = 64, kResultRows = 32;
uint32_t rows_read(int64_t rows) {
  uint32_t n = 8;
  while (n < rows && n < kHalf) n *= 2;
  return n;
}
bool make_map(CUtensorMap* map, const GatedOperand& m, int64_t inner, int64_t outer, uint32_t box_rows, bool bf16) {
  if (m.data == nullptr || reinterpret_cast<uintptr_t>(m.data) % 16 != 0 || m.ld % 8 != 0 || m.ld < inner || inner > 0x7FFFFFFF || outer > 0x7FFFFFFF) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)}, strides[1] = {static_cast<cuuint64_t>(m.ld) * 2};
  const cuuint32_t box[2] = {64, box_rows}, one[2] = {1, 1};
  return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(m.data), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <Out kOut, GatedKeep kKeep>
cudaError_t run(const Work<kMostJobs>& all, int64_t tail, bool high, cudaStream_t s) {
  Work<kJobs<kOut>> w;
  for (int i = 0; i < kJobs<kOut>; ++i) w.job[i] = all.job[i];
  w.f = all.f;
  w.jobs = all.jobs;
  w.items = all.items;
  w.partial = all.partial;
  w.failed = all.failed;
  w.limit = all.limit;
  const auto kernel = gated_kernel<kOut, kKeep>;
  static std::atomic<uint64_t> smem_set{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (!(smem_set.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<kOut>);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(gated_join_kernel<kOut, kKeep>, cudaFuncAttributeMaxDynamicSharedMemorySize, kJoinSmem<kOut, kKeep>);
    if (e != cudaSuccess) return e;
    smem_set.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min(w.items, kPairs)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem<kOut>;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  e = cudaLaunchKernelEx(&cfg, kernel, w);
  if (e != cudaSuccess || tail == 0) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(tail), high ? 2 : 1, (kOut == kActivate ? kHalf : kTile) / kTake<kOut, kKeep>);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = kJoinSmem<kOut, kKeep>;
  note_launch();
  return cudaLaunchKernelEx(&cfg, gated_join_kernel<kOut, kKeep>, w);
}

// A product's maps and shape.
bool make_job(Job& j, const GatedArgs& g, const GatedShape& h) {
  const Sizes z = sizes_of(g.product, h);
  j.a_inner = g.product != GatedProduct::kWeightUp && g.product != GatedProduct::kWeightDown;
  j.b_inner = g.product == GatedProduct::kUp || g.product == GatedProduct::kDown;
  const GatedOperand a[2] = {g.a0, z.results * z.parts > 1 ? g.a1 : g.a0}, b[2] = {g.b0, z.gate || z.parts > 1 ? g.b1 : g.b0};
  const uint32_t a_rows = j.a_inner ? rows_read(z.rows) : kOwnRows;
  j.bytes = 2 * ((j.a_inner ? a_rows * kDepth * 2 : kOperand) + kOperand);
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && a[1].data == a[0].data && a[1].ld == a[0].ld) j.a[1] = j.a[0];
    else if (!make_map(&j.a[i], a[i], j.a_inner ? z.depth : z.rows, j.a_inner ? z.rows : z.depth, a_rows, h.bf16))
      return false;
    if (i == 1 && b[1].data == b[0].data && b[1].ld == b[0].ld) j.b[1] = j.b[0];
    else if (!make_map(&j.b[i], b[i], j.b_inner ? z.depth : z.cols, j.b_inner ? z.cols : z.depth, j.b_inner ? kHalf : kOwnRows, h.bf16))
      return false;
  }
  // h, dg and du have rows of whole groups; the others are a caller's
  const bool between = g.product == GatedProduct::kUp || g.product == GatedProduct::kGate;
  j.to[0] = g.out0;
  j.to[1] = g.out1;
  j.to[2] = g.out2;
  j.rows = z.rows;
  j.cols = between ? gated_pitch(h.hidden) : z.cols;
  j.ldo = between ? j.cols : g.ldo;
  j.wide = j.ldo % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out0) | reinterpret_cast<uintptr_t>(g.out1) | reinterpret_cast<uintptr_t>(g.out2)) % 16 == 0;
  const int results = g.product == GatedProduct::kGate ? 3 : g.product == GatedProduct::kWeightUp ? 2 : 1;
  for (int i = 0; i < 3; ++i) {
    if ((i < results) != (j.to[i] != nullptr)) return false;
    if (i < results && j.wide && !make_map(&j.out[i], {j.to[i], j.ldo}, j.cols, z.rows, kResultRows, h.bf16)) return false;
  }
  return j.wide || !between;
}

}  // namespace

int64_t gated_kept_bytes(const GatedShape& s) {
  const int64_t n = s.tokens * gated_pitch(s.hidden);
  return s.keep == GatedKeep::kNone ? 0 : s.keep == GatedKeep::kWide ? 6 * n : 2 * n + 8 * (n / kGroup8);
}
int64_t gated_partial_bytes(const GatedProduct* p, int n, const GatedShape& s) {
  Plan l[kMostJobs];
  int order[kMostJobs];
  int64_t parts = 0;
  if (n > 1 && plan_together(p, s, n, l, order)) {
    for (int i = 0; i < n; ++i) parts += l[i].tail * l[i].splits;
  } else {
    for (int i = 0; i < n; ++i) {
      plan_one(p[i], s, l[i]);
      parts = std::max(parts, l[i].tail * l[i].splits);
    }
  }
  return parts * kTile * kTile * 4;
}

cudaError_t launch_gated_copies(const GatedCopy* jobs, int n, bool beside, cudaStream_t s) {
  if (n < 1 || n > kGatedCopies) return cudaErrorInvalidValue;
  Copies w{};
  for (int j = 0; j < kGatedCopies; ++j) {
    const bool there = j < n && jobs[j].rows > 0 && jobs[j].cols > 0;
    if (there) w.job[j] = jobs[j];
    w.first[j + 1] = w.first[j] + (there ? ceil_div(jobs[j].rows, kCopyRows) * ceil_div(jobs[j].cols, kCopyCols) : 0);
  }
  const int64_t blocks = w.first[kGatedCopies];
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  note_launch();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kCopyThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gated_copies_kernel, w);
}

cudaError_t launch_gated(const GatedArgs* g, int n, const GatedLaunch& r, cudaStream_t s) {
  const GatedShape& h = r.shape;
  if (n < 1 || n > kMostJobs || h.tokens <= 0 || h.width <= 0 || h.hidden <= 0 || encode_tiled() == nullptr) return cudaErrorInvalidValue;
  // a thread that has made no call of the runtime yet, such as autograd's, has no context, and maps need one
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e != cudaSuccess) return e;
  GatedProduct p[kMostJobs];
  Plan l[kMostJobs];
  int order[kMostJobs];
  for (int i = 0; i < n; ++i) {
    p[i] = g[i].product;
    if (n > 1 && (p[i] == GatedProduct::kUp || p[i] == GatedProduct::kGate)) return cudaErrorInvalidValue;
  }
  if (n == 1) {
    plan_one(p[0], h, l[0]);
    order[0] = 0;
  } else if (!plan_together(p, h, n, l, order)) {
    for (int i = 0; i < n && e == cudaSuccess; ++i) e = launch_gated(g + i, 1, r, s);
    return e;
  }
  Work<kMostJobs> w{};
  int64_t items = 0, parts = 0, joins = 0;
  bool high = false;
  for (int i = 0; i < n; ++i) {
    const Plan& q = l[order[i]];
    Job& j = w.job[i];
    if (!make_job(j, g[order[i]], h) || q.stages > 0x3FFFFFFF) return cudaErrorInvalidValue;
    j.tiles_i = static_cast<int>(q.tiles_i);
    j.tiles_j = static_cast<int>(q.tiles_j);
    j.rows_segment = static_cast<int>(q.tiles_i / (p[order[i]] == GatedProduct::kWeightUp ? 2 : 1));
    j.stages = static_cast<int>(q.stages);
    j.segment = static_cast<int>(q.segment);
    j.first = static_cast<int>(items);
    j.whole = static_cast<int>(q.whole);
    j.splits = static_cast<int>(q.splits);
    j.per_split = static_cast<int>(q.per_split);
    j.part = static_cast<int>(parts);
    j.join = static_cast<int>(joins);
    items += q.whole + q.tail * q.splits;
    parts += q.tail * q.splits;
    joins += q.tail;
    high = high || (q.tail > 0 && j.rows > kHalf);
    if (items + kPairs > 0x7FFFFFFF) return cudaErrorInvalidValue;
  }
  w.jobs = n;
  w.items = static_cast<int>(items);
  w.f.bf16 = h.bf16;
  const double log2e = 1.4426950408889634, gelu = 1.5957691216057308;  // 2 sqrt(2 / pi)
  w.f.curve = h.activation == GatedActivation::kSilu ? Curve{static_cast<float>(-log2e), 0.f}
                                                     : Curve{static_cast<float>(-log2e * gelu), static_cast<float>(-log2e * gelu * 0.044715)};
  w.f.kept = static_cast<char*>(r.kept);
  w.f.rows = h.tokens;
  w.f.pitch = gated_pitch(h.hidden);
  w.partial = r.partial;
  w.failed = r.failed;
  w.limit = r.wait_limit >= 0 ? r.wait_limit : kWaitLimit;
  switch (p[0]) {
    case GatedProduct::kUp:
      switch (h.keep) {
        case GatedKeep::kNone: return run<kActivate, GatedKeep::kNone>(w, joins, high, s);
        case GatedKeep::kWide: return run<kActivate, GatedKeep::kWide>(w, joins, high, s);
        default: return run<kActivate, GatedKeep::kEight>(w, joins, high, s);
      }
    case GatedProduct::kGate:
      return h.keep == GatedKeep::kEight ? run<kDerive, GatedKeep::kEight>(w, joins, high, s) : run<kDerive, GatedKeep::kWide>(w, joins, high, s);
    default: return run<kStore, GatedKeep::kNone>(w, joins, high, s);
  }
}

}  // namespace kern
}  // namespace mccl
