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
constexpr int kStages = 6;
constexpr int kOperand = kHalf * kDepth * 2, kStage = 2 * kOperand;   // bytes a CTA has of a stage
constexpr int kSmem = kStages * kStage + 1024;
constexpr int kColumns = 512;            // of tensor memory: two accumulators
// warp 0 loads, warp 1 issues products, warp 2 has the tensor memory, warps 4 .. 11 take the accumulators out
constexpr int kLoader = 0, kIssuer = 1, kOwner = 2, kFirstOut = 4, kOutWarps = 8, kThreads = 32 * (kFirstOut + kOutWarps);

// ---- PTX ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
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
// Shared-memory matrix descriptors, 128-byte swizzle.  k innermost: rows of 128 bytes (64 k), 1024 bytes per eight rows.  Own
// index innermost: rows of 128 bytes (64 of the index, one k), 1024 bytes per eight k, 8192 from 64 of the index to the next.
template <bool kInner>
__device__ __forceinline__ uint64_t make_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kInner ? 1 : 8192 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// from 16 k to the next, in descriptor units
template <bool kInner>
constexpr uint32_t kStep = (kInner ? 32 : 2048) >> 4;
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
// 32 consecutive columns of the calling thread's lane
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// ... which are there behind this: the operands keep whatever uses them from moving before it.
__device__ __forceinline__ void tmem_wait32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                 "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27])
               :
               : "memory");
  asm volatile("" : "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}

// ---- what a launch is told ----------------------------------------------------------------------------------
enum Out { kStore, kActivate, kDerive };  // what follows the product

struct Finish {
  void *out0, *out1, *out2;
  int64_t ldo;
  bool wide;              // rows of out0 (kStore) may be written 16 bytes at a time
  bool bf16, silu;
  char* kept;
  int64_t rows, cols;     // of one result: tokens x hidden for kActivate and kDerive
  int64_t pitch;          // of h, dg, du
};
struct Work {
  CUtensorMap a[2], b[2];
  Finish f;
  int rows_segment;       // kStore: tiles of rows of the first of two results (dWg, then dWu); all of them where there is one
  int tiles_i, tiles_j;   // tiles_i: of all results
  int stages, segment;    // of the reduction; stages of its first part (dg Wg, then du Wu)
  int whole;              // items that are whole tiles; behind them tiles whose reduction `splits` pairs share
  int items, splits, per_split;
  float* partial;
  uint32_t* failed;
  long long limit;
};

// A tile's place, so that the pairs at work at a time read few rows of each operand: kBand tiles of rows, column by column.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_place(const Work& w, int tile, int& ti, int& tj) {
  const int band = tile / (kBand * w.tiles_j), in_band = tile - band * kBand * w.tiles_j;
  const int high = min(kBand, w.tiles_i - band * kBand);
  tj = in_band / high;
  ti = band * kBand + in_band - tj * high;
}
struct Item {
  int ti, tj, c0, c1, part;  // part: which partial sum, or -1
  __device__ __forceinline__ Item(const Work& w, int item) {
    if (item < w.whole) {
      tile_place(w, item, ti, tj);
      c0 = 0;
      c1 = w.stages;
      part = -1;
    } else {
      part = item - w.whole;
      const int t = part / w.splits;
      tile_place(w, w.whole + t, ti, tj);
      c0 = (part - t * w.splits) * w.per_split;
      c1 = min(w.stages, c0 + w.per_split);
    }
  }
};

// ---- after the product --------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ void store16(void* row, int64_t col, const float* v, bool bf16) {  // 8 numbers
  *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + col) =
      make_uint4(pack2(v[0], v[1], bf16), pack2(v[2], v[3], bf16), pack2(v[4], v[5], bf16), pack2(v[6], v[7], bf16));
}

// s and the slope of act at z.  The exponential and the quotient are within 2^-21 of theirs, which 16 bits do not show.
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
constexpr float kGelu = 1.5957691216057308f, kCubic = 0.044715f;  // 2 sqrt(2 / pi)
__device__ __forceinline__ float gate_of(float z, bool silu) { return logistic(silu ? z : kGelu * (z + kCubic * z * z * z)); }
__device__ __forceinline__ float slope_of(float z, float s, bool silu) {
  const float t = s * (1.f - s);
  // (where the curve is flat the cubic's slope may be infinite)
  return t > 0.f ? s + z * t * (silu ? 1.f : kGelu * (1.f + 3.f * kCubic * z * z)) : s;
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
  k.upper[which][at] = make_uint4(__byte_perm(b[0], b[1], 0x7632), __byte_perm(b[2], b[3], 0x7632), __byte_perm(b[4], b[5], 0x7632),
                                  __byte_perm(b[6], b[7], 0x7632));
  k.lower[which][at] = make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0051), __byte_perm(b[2], b[3], 0x0051), 0x5410),
                                  __byte_perm(__byte_perm(b[4], b[5], 0x0051), __byte_perm(b[6], b[7], 0x0051), 0x5410));
}
__device__ __forceinline__ void take_wide(const uint4& up, const uint2& low, float* v) {
  const uint32_t u[4] = {up.x, up.y, up.z, up.w}, l[2] = {low.x, low.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t high = i % 2 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16;
    v[i] = __uint_as_float(high | ((l[i / 4] >> (8 * (i % 4))) & 0xFFu) << 8);
  }
}

// Columns col .. col + kN of a row of a result.
template <int kN>
__device__ __forceinline__ void finish_store(const Finish& f, void* out, int64_t rows, int64_t row, int64_t col, const float* v) {
  if (row >= rows || col >= f.cols) return;
  uint16_t* to = static_cast<uint16_t*>(out) + row * f.ldo;
  if (f.wide && col + kN <= f.cols) {
#pragma unroll
    for (int i = 0; i < kN; i += 8) store16(to, col + i, v + i, f.bf16);
  } else {
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const uint32_t p = pack2(v[i], v[i + 1], f.bf16);
      if (col + i < f.cols) to[col + i] = static_cast<uint16_t>(p);
      if (col + i + 1 < f.cols) to[col + i + 1] = static_cast<uint16_t>(p >> 16);
    }
  }
}
// kN columns of g and u to h and to what is kept.
template <GatedKeep kKeep, int kN>
__device__ __forceinline__ void finish_activate(const Finish& f, int64_t row, int64_t col, const float* g, const float* u) {
  if (row >= f.rows || col >= f.pitch) return;
  if constexpr (kKeep == GatedKeep::kEight) {
    static_assert(kN == kGroup8, "a thread has a whole group");
    const Eight k(f.kept, f.rows, f.pitch);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float* v = which ? u : g;
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < kN; ++i) most = most8(most, v[i]);
      const Scale8 s = scale8(most);
      k.scales[which][col / kGroup8 * f.rows + row] = s.scale;
#pragma unroll
      for (int i = 0; i < kN; i += 16)
        k.codes[which][(col + i) / 16 * f.rows + row] =
            make_uint4(codes8(v[i], v[i + 1], v[i + 2], v[i + 3], s.inverse), codes8(v[i + 4], v[i + 5], v[i + 6], v[i + 7], s.inverse),
                       codes8(v[i + 8], v[i + 9], v[i + 10], v[i + 11], s.inverse), codes8(v[i + 12], v[i + 13], v[i + 14], v[i + 15], s.inverse));
    }
  }
  uint16_t* to = static_cast<uint16_t*>(f.out0) + row * f.pitch;
#pragma unroll
  for (int i = 0; i < kN; i += 8) {
    if constexpr (kKeep == GatedKeep::kWide) {
      const Wide k(f.kept, f.rows, f.pitch);
      const int64_t at = (col + i) / 8 * f.rows + row;
      keep_wide(k, 0, at, g + i);
      keep_wide(k, 1, at, u + i);
    }
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = g[i + e] * gate_of(g[i + e], f.silu) * u[i + e];
    store16(to, col + i, h, f.bf16);
  }
}
// kN columns (a multiple of 16) of dh to h, dg and du.
template <GatedKeep kKeep, int kN>
__device__ __forceinline__ void finish_derive(const Finish& f, int64_t row, int64_t col, const float* dh) {
  if (row >= f.rows || col >= f.pitch) return;
  const int64_t to = row * f.pitch;
  float scale[2];
  if constexpr (kKeep == GatedKeep::kEight) {
    const Eight k(f.kept, f.rows, f.pitch);
#pragma unroll
    for (int which = 0; which < 2; ++which) scale[which] = k.scales[which][col / kGroup8 * f.rows + row];
  }
#pragma unroll
  for (int i = 0; i < kN; i += 16) {
    float z[2][16];
    if constexpr (kKeep == GatedKeep::kEight) {
      const Eight k(f.kept, f.rows, f.pitch);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint4 c = __ldcs(k.codes[which] + (col + i) / 16 * f.rows + row);
        const uint32_t words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int e = 0; e < 16; ++e) z[which][e] = value8(words[e / 4], e % 4, scale[which]);
      }
    } else {
      const Wide k(f.kept, f.rows, f.pitch);
#pragma unroll
      for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int64_t at = ((col + i) / 8 + b) * f.rows + row;
          take_wide(__ldcs(k.upper[which] + at), __ldcs(k.lower[which] + at), &z[which][8 * b]);
        }
    }
#pragma unroll
    for (int b = 0; b < 16; b += 8) {
      float h[8], dg[8], du[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float g = z[0][b + e], u = z[1][b + e], d = dh[i + b + e];
        const float s = gate_of(g, f.silu), a = g * s;
        h[e] = a * u;
        du[e] = d * a;
        dg[e] = d * u * slope_of(g, s, f.silu);
      }
      store16(static_cast<uint16_t*>(f.out0) + to, col + i + b, h, f.bf16);
      store16(static_cast<uint16_t*>(f.out1) + to, col + i + b, dg, f.bf16);
      store16(static_cast<uint16_t*>(f.out2) + to, col + i + b, du, f.bf16);
    }
  }
}

// ---- product ------------------------------------------------------------------------------------------------
// The columns that a thread takes at a time: of h for kActivate (two accumulator columns each), of c else.
template <Out kOut, GatedKeep kKeep>
constexpr int kTake = kOut == kActivate && kKeep == GatedKeep::kEight ? 64 : 32;

template <Out kOut, GatedKeep kKeep, typename Fetch>
__device__ __forceinline__ void finish_tile(const Work& w, int ti, int tj, int row_in_tile, int first, int last, const Fetch& fetch) {
  constexpr int kN = kTake<kOut, kKeep>;
  const Finish& f = w.f;
#pragma unroll 1
  for (int c = first; c < last; c += kN) {
    if constexpr (kOut == kActivate) {
      float g[kN], u[kN];
      fetch(c, g);
      fetch(kHalf + c, u);
      finish_activate<kKeep, kN>(f, static_cast<int64_t>(ti) * kTile + row_in_tile, static_cast<int64_t>(tj) * kHalf + c, g, u);
    } else {
      float v[kN];
      fetch(c, v);
      if constexpr (kOut == kDerive) {
        finish_derive<kKeep, kN>(f, static_cast<int64_t>(ti) * kTile + row_in_tile, static_cast<int64_t>(tj) * kTile + c, v);
      } else {
        const bool second = ti >= w.rows_segment;
        finish_store<kN>(f, second ? f.out1 : f.out0, f.rows, static_cast<int64_t>(second ? ti - w.rows_segment : ti) * kTile + row_in_tile,
                         static_cast<int64_t>(tj) * kTile + c, v);
      }
    }
  }
}

// A pair of CTAs per tile of 256 x 256, tiles in turn: each CTA loads half of either operand's rows and has half of the
// accumulator's; the first one issues the products of both.  Two accumulators, so that a tile is taken out while the next one
// is multiplied.
template <bool kAInner, bool kBInner, Out kOut, GatedKeep kKeep>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gated_kernel(const __grid_constant__ Work w) {
  extern __shared__ char raw[];
  __shared__ alignas(8) uint64_t bars[2 * kStages + 5];
  __shared__ uint32_t tmem_base;
  const uint32_t smem0 = (smem_addr(raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const uint32_t bar0 = smem_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
  auto acc_free = [&](int b) { return bar0 + 8u * (2 * kStages + 2 + b); };
  const uint32_t drained = bar0 + 8u * (2 * kStages + 4);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
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
  asm volatile("griddepcontrol.wait;" ::: "memory");
  bool ok = true, issued = false;

  if (warp == kLoader) {
    if (elect()) {
      int s = 0, turn = 0;
      for (int item = pair; ok && item < w.items; item += pairs) {
        const Item t(w, item);
        const int i_second = t.ti >= w.rows_segment, i0 = (i_second ? t.ti - w.rows_segment : t.ti) * kTile + rank * kHalf;
        // g and u side by side: one CTA has the rows of Wg, the other those of Wu
        const int j0 = kOut == kActivate ? t.tj * kHalf : t.tj * kTile + rank * kHalf;
        for (int c = t.c0; ok && c < t.c1; ++c) {
          ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
          if (!ok) break;
          const int k_second = c >= w.segment, k0 = (k_second ? c - w.segment : c) * kDepth;
          const CUtensorMap* a = &w.a[i_second | k_second];
          const CUtensorMap* b = &w.b[kOut == kActivate ? rank : k_second];
          const uint32_t to = smem0 + s * kStage, bar = in_leader(full(s));
          if (rank == 0) bar_expect(full(s), 2 * kStage);
          if (kAInner) load_box(to, a, k0, i0, bar);
          else {
            load_box(to, a, i0, k0, bar);
            load_box(to + kOperand / 2, a, i0 + 64, k0, bar);
          }
          if (kBInner) load_box(to + kOperand, b, k0, j0, bar);
          else {
            load_box(to + kOperand, b, j0, k0, bar);
            load_box(to + kOperand + kOperand / 2, b, j0 + 64, k0, bar);
          }
          if (++s == kStages) s = 0, ++turn;
        }
      }
      // the products' last arrivals, before the barriers are another's
      for (int left = 0; ok && left < kStages; ++left) {
        ok = bar_wait(empty(s), (turn & 1) ^ 1, w.limit);
        if (++s == kStages) s = 0, ++turn;
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    if (rank == 0 && elect()) {
      issued = true;
      ok = w.limit > 0;  // a limit of zero, of tests: no product is issued, and all others wait in vain
      const uint32_t idesc = make_idesc(w.f.bf16, kAInner, kBInner);
      const uint64_t a0 = make_desc<kAInner>(smem0), b0 = make_desc<kBInner>(smem0 + kOperand);
      int s = 0, turn = 0, done = 0;
      for (int item = pair; ok && item < w.items; item += pairs, ++done) {
        const Item t(w, item);
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
          for (int k = 0; k < kDepth / 16; ++k) mma(acc, a + k * kStep<kAInner>, b + k * kStep<kBInner>, idesc, c > t.c0 || k > 0);
          mma_commit(empty(s));
          if (++s == kStages) s = 0, ++turn;
        }
        if (ok) mma_commit(acc_full(buffer));
      }
    }
    __syncwarp();
  } else if (warp >= kFirstOut) {
    // lanes 32 q .. 32 q + 31 of tensor memory are open to the warps with warp % 4 == q; two of them share the columns
    const int q = warp & 3, half = (warp - kFirstOut) >> 2;
    const int row = rank * kHalf + 32 * q + lane;
    constexpr int kShare = (kOut == kActivate ? kHalf : kTile) / 2;
    int done = 0;
    for (int item = pair; item < w.items; item += pairs, ++done) {
      const Item t(w, item);
      const int buffer = done & 1;
      if (ok) ok = __all_sync(0xFFFFFFFFu, bar_wait(acc_full(buffer), (done >> 1) & 1, w.limit));
      fence_after();
      const uint32_t from = tmem + buffer * kTile + (static_cast<uint32_t>(32 * q) << 16);
      auto fetch = [&](int c, float* v) {
        constexpr int kN = kTake<kOut, kKeep>;
        if (ok) {
#pragma unroll
          for (int i = 0; i < kN; i += 32) tmem_load32(from + c + i, v + i);
#pragma unroll
          for (int i = 0; i < kN; i += 32) tmem_wait32(v + i);
        } else {
#pragma unroll
          for (int i = 0; i < kN; ++i) v[i] = NAN;  // no number that looks like a result
        }
      };
      if (t.part < 0) {
        finish_tile<kOut, kKeep>(w, t.ti, t.tj, row, half * kShare, half * kShare + kShare, fetch);
      } else {
        const bool second = t.ti >= w.rows_segment;
        const bool there = static_cast<int64_t>(second ? t.ti - w.rows_segment : t.ti) * kTile + row < w.f.rows;
        float* to = w.partial + static_cast<int64_t>(t.part) * (kTile * kTile) + row;
#pragma unroll 1
        for (int c = half * kHalf; c < half * kHalf + kHalf; c += 32) {
          float v[kTake<kOut, kKeep>];
          if (ok) {
            tmem_load32(from + c, v);
            tmem_wait32(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = NAN;
          }
          if (there)
#pragma unroll
            for (int i = 0; i < 32; ++i) __stcg(to + static_cast<int64_t>(c + i) * kTile, v[i]);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0 && ok) bar_arrive_cluster(in_leader(acc_free(buffer)));
    }
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

// Adds up the parts of the tiles whose reduction was shared, in order, and finishes them.  A block has 32 (64) columns of half a
// tile; a part is read in runs of 128 numbers.
template <Out kOut, GatedKeep kKeep>
__global__ void __launch_bounds__(kHalf) gated_join_kernel(const __grid_constant__ Work w) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kN = kTake<kOut, kKeep>;
  const int tile = blockIdx.x, first = blockIdx.z * kN, row = blockIdx.y * kHalf + threadIdx.x;
  int ti, tj;
  tile_place(w, w.whole + tile, ti, tj);
  if (static_cast<int64_t>(ti >= w.rows_segment ? ti - w.rows_segment : ti) * kTile + row >= w.f.rows) return;
  const float* from = w.partial + static_cast<int64_t>(tile) * w.splits * (kTile * kTile) + row;
  auto fetch = [&](int c, float* v) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = 0.f;
    for (int p = 0; p < w.splits; ++p) {
      const float* x = from + static_cast<int64_t>(p) * (kTile * kTile) + static_cast<int64_t>(c) * kTile;
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] += __ldcg(x + i * kTile);
    }
  };
  finish_tile<kOut, kKeep>(w, ti, tj, row, first, first + kN, fetch);
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
  int64_t whole, tail, splits, per_split;
};
// Whole tiles as long as they fill the device; the rest, less than one tile a pair, is shared along the reduction where
// that saves more than the partial sums and their launch cost.
Plan plan_of(GatedProduct p, const GatedShape& s) {
  const Sizes z = sizes_of(p, s);
  Plan l{};
  l.tiles_i = ceil_div(z.rows, kTile) * z.results;
  l.tiles_j = ceil_div(z.cols, z.gate ? kHalf : kTile);
  l.segment = ceil_div(z.depth, kDepth);
  l.stages = l.segment * z.parts;
  const int64_t tiles = l.tiles_i * l.tiles_j;
  l.tail = tiles % kPairs;
  l.whole = tiles - l.tail;
  l.splits = 1;
  l.per_split = l.stages;
  if (l.tail > 0) {
    const int64_t most = std::min<int64_t>({kPairs / l.tail, l.stages / 4, 16});
    if (most >= 2) {
      const int64_t per = ceil_div(l.stages, most), splits = ceil_div(l.stages, per);
      // microseconds: a stage takes 0.37; a partial sum is written and read at 4 TB/s, behind 4 for the launch
      const double saved = 0.37 * static_cast<double>(l.stages - per);
      const double cost = 4.0 + 8.0 * static_cast<double>(l.tail * splits * kTile * std::min<int64_t>(kTile, z.rows)) / 4e6;
      if (saved > cost) {
        l.splits = splits;
        l.per_split = per;
      }
    }
  }
  if (l.splits == 1) {
    l.whole = tiles;
    l.tail = 0;
  }
  return l;
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
// A matrix of `outer` rows of `inner` numbers; boxes of 64 of a row, and of 128 rows (k innermost) or 64 (own index innermost).
bool make_map(CUtensorMap* map, const GatedOperand& m, int64_t inner, int64_t outer, bool k_inner, bool bf16) {
  if (m.data == nullptr || reinterpret_cast<uintptr_t>(m.data) % 16 != 0 || m.ld % 8 != 0 || m.ld < inner || inner > 0x7FFFFFFF || outer > 0x7FFFFFFF) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)}, strides[1] = {static_cast<cuuint64_t>(m.ld) * 2};
  const cuuint32_t box[2] = {64, k_inner ? 128u : 64u}, one[2] = {1, 1};
  return encode_tiled()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(m.data), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kAInner, bool kBInner, Out kOut, GatedKeep kKeep>
cudaError_t run(const Work& w, int64_t tail, cudaStream_t s) {
  const auto kernel = gated_kernel<kAInner, kBInner, kOut, kKeep>;
  static std::atomic<uint64_t> smem_set{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (!(smem_set.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    smem_set.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(std::min(w.items, kPairs)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  e = cudaLaunchKernelEx(&cfg, kernel, w);
  if (e != cudaSuccess || tail == 0) return e;
  constexpr int kN = kTake<kOut, kKeep>;
  cfg.gridDim = dim3(static_cast<unsigned>(tail), w.f.rows > kHalf ? 2 : 1, (kOut == kActivate ? kHalf : kTile) / kN);
  cfg.blockDim = dim3(kHalf);
  cfg.dynamicSmemBytes = 0;
  note_launch();
  return cudaLaunchKernelEx(&cfg, gated_join_kernel<kOut, kKeep>, w);
}

}  // namespace

int64_t gated_kept_bytes(const GatedShape& s) {
  const int64_t n = s.tokens * gated_pitch(s.hidden);
  return s.keep == GatedKeep::kNone ? 0 : s.keep == GatedKeep::kWide ? 6 * n : 2 * n + 8 * (n / kGroup8);
}
int64_t gated_partial_bytes(GatedProduct p, const GatedShape& s) {
  const Plan l = plan_of(p, s);
  return l.tail * l.splits * kTile * kTile * 4;
}

cudaError_t launch_gated(const GatedArgs& g, cudaStream_t s) {
  const GatedShape& h = g.shape;
  if (h.tokens <= 0 || h.width <= 0 || h.hidden <= 0 || encode_tiled() == nullptr) return cudaErrorInvalidValue;
  const Sizes z = sizes_of(g.product, h);
  const Plan l = plan_of(g.product, h);
  if (l.tiles_i * l.tiles_j * 16 + 1 > 0x7FFFFFFF || z.depth > 0x3FFFFFFF) return cudaErrorInvalidValue;
  // a thread that has made no call of the runtime yet, such as autograd's, has no context, and maps need one
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e != cudaSuccess) return e;
  Work w{};
  const bool a_inner = g.product != GatedProduct::kWeightUp && g.product != GatedProduct::kWeightDown;
  const bool b_inner = g.product == GatedProduct::kUp || g.product == GatedProduct::kDown;
  const GatedOperand a[2] = {g.a0, z.results * z.parts > 1 ? g.a1 : g.a0}, b[2] = {g.b0, z.gate || z.parts > 1 ? g.b1 : g.b0};
  for (int i = 0; i < 2; ++i)
    if (!make_map(&w.a[i], a[i], a_inner ? z.depth : z.rows, a_inner ? z.rows : z.depth, a_inner, h.bf16) ||
        !make_map(&w.b[i], b[i], b_inner ? z.depth : z.cols, b_inner ? z.cols : z.depth, b_inner, h.bf16))
      return cudaErrorInvalidValue;
  w.f.out0 = g.out0;
  w.f.out1 = g.out1;
  w.f.out2 = g.out2;
  w.f.ldo = g.ldo;
  w.f.wide = g.ldo % 8 == 0 && (reinterpret_cast<uintptr_t>(g.out0) | reinterpret_cast<uintptr_t>(g.out1)) % 16 == 0;
  w.f.bf16 = h.bf16;
  w.f.silu = h.activation == GatedActivation::kSilu;
  w.f.kept = static_cast<char*>(g.kept);
  w.f.rows = z.rows;
  w.f.cols = z.cols;
  w.f.pitch = gated_pitch(h.hidden);
  w.tiles_i = static_cast<int>(l.tiles_i);
  w.tiles_j = static_cast<int>(l.tiles_j);
  w.rows_segment = static_cast<int>(l.tiles_i / z.results);
  w.stages = static_cast<int>(l.stages);
  w.segment = static_cast<int>(l.segment);
  w.whole = static_cast<int>(l.whole);
  w.splits = static_cast<int>(l.splits);
  w.per_split = static_cast<int>(l.per_split);
  w.items = static_cast<int>(l.whole + l.tail * l.splits);
  w.partial = g.partial;
  w.failed = g.failed;
  w.limit = g.wait_limit >= 0 ? g.wait_limit : kWaitLimit;
  switch (g.product) {
    case GatedProduct::kUp:
      switch (h.keep) {
        case GatedKeep::kNone: return run<true, true, kActivate, GatedKeep::kNone>(w, l.tail, s);
        case GatedKeep::kWide: return run<true, true, kActivate, GatedKeep::kWide>(w, l.tail, s);
        default: return run<true, true, kActivate, GatedKeep::kEight>(w, l.tail, s);
      }
    case GatedProduct::kDown: return run<true, true, kStore, GatedKeep::kNone>(w, l.tail, s);
    case GatedProduct::kGate:
      return h.keep == GatedKeep::kEight ? run<true, false, kDerive, GatedKeep::kEight>(w, l.tail, s)
                                         : run<true, false, kDerive, GatedKeep::kWide>(w, l.tail, s);
    case GatedProduct::kInput: return run<true, false, kStore, GatedKeep::kNone>(w, l.tail, s);
    default: return run<false, false, kStore, GatedKeep::kNone>(w, l.tail, s);
  }
}

}  // namespace kern
}  // namespace mccl
