// Norms of queries and keys for each head, with the rotation by position in the same pass, and its gradients (sm_100a).
//
// Of a row x of D: r = 1 / sqrt(mean(x^2) + eps), n = x r w; the first R numbers of n are R / 2 pairs (a, b), rotated by the
// token's angles: a' = a c - b s, b' = b c + a s.  Backward, with dn the gradient rotated back:
//     dw = sum over rows of dn x r        dx = r (dn w - x r^2 mean(dn w x))
// r is computed again from x, which backward reads anyway.  All of it in fp32, rounded once.
//
// Bound by memory.  A team of lanes, 8 pairs each, has a row in registers; both members of a pair are in the same lane, so the
// rotation moves nothing between lanes and the norm is the only sum over a team.  A team takes several heads of its token, for
// which the angles stay in registers.  32768 tokens of 40 heads of 128, bf16: forward 129 us (5.2 TB/s), backward, values copied, 262
// (4.4); 8192 tokens of 32 heads of 64 15 and 37 us (B200; 4.6 and 3.6 TB/s).  Backward half of the issue slots are busy, half of the
// time for want of numbers: its two rows and two gradients a lane in flight are what 128 registers hold; each is asked for again as
// soon as its numbers are used, the next token's at a token's end (269 us when both were waited for together).  Forward, with four
// rows, that gains nothing and costs 2 us of 8192 tokens.  Sums of two numbers by one instruction: 137 and 273 us.
#include <algorithm>
#include <type_traits>

#include "kernels/elems.cuh"
#include "kernels/heads_api.h"
#include "kernels/launch_count.h"

namespace mccl {
namespace kern {
namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;
constexpr int kForwardResident = 2, kBackwardResident = 2;  // blocks an SM, for their registers
constexpr int kCopies = 4;                                   // rows of values in flight

// Queries, keys and (backward, one gradient for all three) values are sides with blocks of their own: a thread then has one
// weight and one gradient of it in registers (with both it took 223 of them backward, one block an SM).
struct Side {
  HeadRows x, dy;         // what is read; forward, and for values, one of them
  char* out;
  int64_t out_token;      // elements from one token's rows to the next
  const void* weight;
  int heads;
  int parts;              // teams that share a token's heads: 2^parts
  int64_t units;          // tokens x 2^parts
  int first, blocks;      // of the grid
};
struct Plan {
  Side side[3];
  int sides, team, blocks;  // team: lanes that share a row, a power of two
};

// The pairs of a lane: `at` and `at2` are where the first members and the second members begin.  Halves: the rotated pairs are
// (i, i + R/2), the rest is paired alike, so that both members' runs are contiguous.  Neighbours: pairs (2 i, 2 i + 1).
template <int V, bool kNear>
struct Lane {
  int pair, at, at2, n, n2;  // n, n2: how many of each exist
  bool rotated;
  __device__ __forceinline__ Lane(const HeadsShape& s, int lane, int run) {
    const int half = s.rotary / 2, rest = (s.dim - s.rotary + 1) / 2;
    pair = (lane + run) * V;
    rotated = pair < half;
    if (kNear) {
      at = 2 * pair;
      at2 = at + V;
      n = min(max(s.dim - at, 0), V);
      n2 = min(max(s.dim - at2, 0), V);
    } else if (rotated) {
      at = pair;
      at2 = pair + half;
      n = n2 = V;  // host: V divides R / 2
    } else {
      const int p = pair - half;
      at = s.rotary + p;
      at2 = at + rest;
      n = p < rest ? min(V, s.dim - at) : 0;
      n2 = p < rest ? min(max(s.dim - at2, 0), V) : 0;
    }
  }
};

// A lane's pairs as they lie in memory: two runs of V numbers.  A run of four or eight is there whole or not at all (run_of).
template <typename T, int V>
using RunOf = std::conditional_t<V == 1, T, std::conditional_t<V * sizeof(T) == 8, uint2, uint4>>;

template <typename T, int V, bool kNear>
struct Pairs {
  using Raw = RunOf<T, V>;
  Raw run[2];
  __device__ __forceinline__ void load(const T* row, const Lane<V, kNear>& l, bool on) {
    run[0] = on && l.n > 0 ? *reinterpret_cast<const Raw*>(row + l.at) : Raw{};
    run[1] = on && l.n2 > 0 ? *reinterpret_cast<const Raw*>(row + l.at2) : Raw{};
  }
  __device__ __forceinline__ void store(T* row, const Lane<V, kNear>& l, bool on) const {
    if (on && l.n > 0) *reinterpret_cast<Raw*>(row + l.at) = run[0];
    if (on && l.n2 > 0) *reinterpret_cast<Raw*>(row + l.at2) = run[1];
  }
  // the members of pair i
  __device__ __forceinline__ float a(int i) const { return kNear ? get(2 * i) : get(i); }
  __device__ __forceinline__ float b(int i) const { return kNear ? get(2 * i + 1) : get(V + i); }
  __device__ __forceinline__ void set(const float (&a)[V], const float (&b)[V]) {
    float v[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[kNear ? 2 * i : i] = a[i];
      v[kNear ? 2 * i + 1 : V + i] = b[i];
    }
    run[0] = pack_run<T, V, Raw>(v);
    run[1] = pack_run<T, V, Raw>(v + V);
  }

 private:
  __device__ __forceinline__ float get(int i) const { return Traits<T>::load(reinterpret_cast<const T*>(&run[i / V])[i % V]); }
};

// The lane's weights, element by element unless they are fp32 in aligned runs.
template <typename T, int V, bool kNear>
__device__ __forceinline__ void load_weight(const void* w, bool f32, const Lane<V, kNear>& l, float (&a)[V], float (&b)[V]) {
  if constexpr (V > 1) {
    if (f32 && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
      float v[2 * V];
      load_run<float, V>(static_cast<const float*>(w) + l.at, l.n, l.n > 0, *reinterpret_cast<float(*)[V]>(v));
      load_run<float, V>(static_cast<const float*>(w) + l.at2, l.n2, l.n2 > 0, *reinterpret_cast<float(*)[V]>(v + V));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[i] = v[kNear ? 2 * i : i];
        b[i] = v[kNear ? 2 * i + 1 : V + i];
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int ia = kNear ? l.at + 2 * i : l.at + i, ib = kNear ? ia + 1 : l.at2 + i;
    const bool ha = kNear ? ia < l.at + l.n + l.n2 : i < l.n, hb = kNear ? ib < l.at + l.n + l.n2 : i < l.n2;
    a[i] = !ha ? 0.f : f32 ? static_cast<const float*>(w)[ia] : Traits<T>::load(static_cast<const T*>(w)[ia]);
    b[i] = !hb ? 0.f : f32 ? static_cast<const float*>(w)[ib] : Traits<T>::load(static_cast<const T*>(w)[ib]);
  }
}

// Cosines and sines of a lane's pairs, which are rotated.
template <int V>
__device__ __forceinline__ void load_angles(const HeadsShape& s, int64_t position, int pair, float (&c)[V], float (&n)[V]) {
  const bool inside = position >= 0 && position < s.table_rows;
  const float* row = s.table + (inside ? position : 0) * s.rotary + pair;
  if (inside) {
    load_run<float, V>(row, V, true, c);
    load_run<float, V>(row + s.rotary / 2, V, true, n);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) c[i] = n[i] = NAN;
  }
}

__device__ __forceinline__ int64_t position_of(const HeadsShape& s, int64_t b, int64_t t) {
  if (s.positions == nullptr) return t;
  const int64_t i = b * s.pos_batch + t * s.pos_token;
  return s.positions_32 ? static_cast<const int32_t*>(s.positions)[i] : static_cast<const int64_t*>(s.positions)[i];
}
__device__ __forceinline__ float team_sum(float v, int team) {
  for (int m = team / 2; m > 0; m /= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
  return v;
}

// What a block's threads are about: their side, their team's units.
struct Walk {
  int side, lane;
  int64_t teams, base, step, mine;
  __device__ __forceinline__ explicit Walk(const Plan& w) {
    side = 0;
    while (side + 1 < w.sides && static_cast<int>(blockIdx.x) >= w.side[side + 1].first) ++side;
    lane = threadIdx.x % w.team;
    mine = threadIdx.x / w.team;
    teams = kThreads / w.team;
    base = (static_cast<int>(blockIdx.x) - w.side[side].first) * teams;
    step = w.side[side].blocks * teams;
  }
};
struct Token {
  int64_t at, b, t;
  int first;  // head
  bool there;
  __device__ __forceinline__ Token(const Side& d, const HeadsShape& s, int64_t unit) {
    there = unit < d.units;
    if (!there) unit = 0;
    at = unit >> d.parts;
    first = static_cast<int>(unit) & ((1 << d.parts) - 1);
    if (s.batches == 1) b = 0;
    else if (d.units <= 0xFFFFFFFFll) b = static_cast<uint32_t>(at) / static_cast<uint32_t>(s.tokens);  // no more tokens than units
    else b = at / s.tokens;
    t = at - b * s.tokens;
  }
};
template <typename T>
__device__ __forceinline__ const T* token_rows(const HeadRows& r, const Token& k) {
  return static_cast<const T*>(r.data) + k.b * r.batch + k.t * r.token;
}

// kRows rows of each team are in flight before the first is used: the first of a token before its angles are asked for, the next
// ones while the results leave.  Weights and angles become one factor for each member of a pair in each result.
template <typename T, int V, int K, bool kNear, int kRows>
__global__ void __launch_bounds__(kThreads, V > 1 && K == 1 ? kForwardResident : 1) heads_forward_kernel(const HeadsShape s, const Plan w) {
  const Walk walk(w);
  const Side& d = w.side[walk.side];
  const int lane = walk.lane, step = 1 << d.parts;
  const float inv = 1.f / static_cast<float>(s.dim);
  for (int64_t base = walk.base; base < d.units; base += walk.step) {
    const Token token(d, s, base + walk.mine);
    const T* from = token_rows<T>(d.x, token);
    Pairs<T, V, kNear> x[kRows][K];
    auto load = [&](int h0) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int h = h0 + j * step + token.first;
#pragma unroll
        for (int k = 0; k < K; ++k) x[j][k].load(from + h * d.x.head, Lane<V, kNear>(s, lane, k * w.team), token.there && h < d.heads);
      }
    };
    load(0);
    const int64_t position = position_of(s, token.b, token.t);
    float fa[K][2][V], fb[K][2][V];  // of a in a' and b', of b in b' and a'
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Lane<V, kNear> l(s, lane, k * w.team);
      load_weight<T>(d.weight, s.weights_f32, l, fa[k][0], fb[k][0]);
      if (l.rotated) {
        float c[V], n[V];
        load_angles<V>(s, position, l.pair, c, n);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          fa[k][1][i] = fa[k][0][i] * n[i];
          fb[k][1][i] = -fb[k][0][i] * n[i];
          fa[k][0][i] *= c[i];
          fb[k][0][i] *= c[i];
        }
      }
    }
    T* to = reinterpret_cast<T*>(d.out) + token.at * d.out_token;
    for (int h0 = 0; h0 < d.heads; h0 += kRows * step) {
      if (h0 > 0) load(h0);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int h = h0 + j * step + token.first;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) sum += x[j][k].a(i) * x[j][k].a(i) + x[j][k].b(i) * x[j][k].b(i);
        const float r = rsqrtf(team_sum(sum, w.team) * inv + s.eps);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const Lane<V, kNear> l(s, lane, k * w.team);
          float na[V], nb[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float a = x[j][k].a(i) * r, b = x[j][k].b(i) * r;
            na[i] = a * fa[k][0][i];
            nb[i] = b * fb[k][0][i];
            if (l.rotated) {
              na[i] += b * fb[k][1][i];
              nb[i] += a * fa[k][1][i];
            }
          }
          Pairs<T, V, kNear> y;
          y.set(na, nb);
          y.store(to + static_cast<int64_t>(h) * s.dim, l, token.there && h < d.heads);
        }
      }
    }
  }
}

// The gradients of the weights: each lane adds up its columns over all of its rows, the block's teams are joined in shared
// memory, and heads_weights_kernel adds the blocks, all in a fixed order.
template <typename T, int V, int K, bool kNear, int kRows>
__global__ void __launch_bounds__(kThreads, V > 1 && K == 1 ? kBackwardResident : 1) heads_backward_kernel(const HeadsShape s, const Plan w, float* __restrict__ partial) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // heads_weights_kernel, which waits for all of this
  const Walk walk(w);
  const Side& d = w.side[walk.side];
  const int lane = walk.lane, step = 1 << d.parts;
  if (walk.side == 2) {  // values: their gradient goes to its place
    for (int64_t base = walk.base; base < d.units; base += walk.step) {
      const Token token(d, s, base + walk.mine);
      const T* from = token_rows<T>(d.x, token);
      T* to = reinterpret_cast<T*>(d.out) + token.at * d.out_token;
      for (int h0 = token.first; h0 < d.heads && token.there; h0 += kCopies * step) {
        Pairs<T, V, kNear> x[kCopies][K];
#pragma unroll
        for (int j = 0; j < kCopies; ++j)
#pragma unroll
          for (int k = 0; k < K; ++k) x[j][k].load(from + (h0 + j * step) * d.x.head, Lane<V, kNear>(s, lane, k * w.team), h0 + j * step < d.heads);
#pragma unroll
        for (int j = 0; j < kCopies; ++j)
#pragma unroll
          for (int k = 0; k < K; ++k)
            x[j][k].store(to + static_cast<int64_t>(h0 + j * step) * s.dim, Lane<V, kNear>(s, lane, k * w.team), h0 + j * step < d.heads);
      }
    }
    return;
  }
  float grad[K][2][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) grad[k][0][i] = grad[k][1][i] = 0.f;
  const float inv = 1.f / static_cast<float>(s.dim);
  Pairs<T, V, kNear> x[kRows][K], g[kRows][K];
  auto load = [&](int j, const T* xs, const T* gs, int h, bool there) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Lane<V, kNear> l(s, lane, k * w.team);
      x[j][k].load(xs + h * d.x.head, l, there && h < d.heads);
      g[j][k].load(gs + h * d.dy.head, l, there && h < d.heads);
    }
  };
  Token next(d, s, walk.base + walk.mine);
  const T *next_from = token_rows<T>(d.x, next), *next_gfrom = token_rows<T>(d.dy, next);
#pragma unroll
  for (int j = 0; j < kRows; ++j) load(j, next_from, next_gfrom, j * step + next.first, next.there);
  for (int64_t base = walk.base; base < d.units; base += walk.step) {
    const Token token = next;
    const T *from = next_from, *gfrom = next_gfrom;
    next = Token(d, s, base + walk.step + walk.mine);
    next_from = token_rows<T>(d.x, next);
    next_gfrom = token_rows<T>(d.dy, next);
    const int64_t position = position_of(s, token.b, token.t);
    float weight[K][2][V], c[K][V], sn[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Lane<V, kNear> l(s, lane, k * w.team);
      load_weight<T>(d.weight, s.weights_f32, l, weight[k][0], weight[k][1]);
      if (l.rotated) load_angles<V>(s, position, l.pair, c[k], sn[k]);
    }
    T* to = reinterpret_cast<T*>(d.out) + token.at * d.out_token;
    for (int h0 = 0; h0 < d.heads; h0 += kRows * step) {
      const bool more = h0 + kRows * step < d.heads;
      const T *then = more ? from : next_from, *gthen = more ? gfrom : next_gfrom;
      const int then_h = more ? h0 + kRows * step + token.first : next.first;
      const bool then_there = more ? token.there : next.there;
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int h = h0 + j * step + token.first;
        const bool on = token.there && h < d.heads;
        float sum = 0.f, dot = 0.f, na[K][V], nb[K][V];  // the gradient rotated back
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const Lane<V, kNear> l(s, lane, k * w.team);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float ga = g[j][k].a(i), gb = g[j][k].b(i), xa = x[j][k].a(i), xb = x[j][k].b(i);
            na[k][i] = l.rotated ? ga * c[k][i] + gb * sn[k][i] : ga;
            nb[k][i] = l.rotated ? gb * c[k][i] - ga * sn[k][i] : gb;
            sum += xa * xa + xb * xb;
            dot += (na[k][i] * weight[k][0][i]) * xa + (nb[k][i] * weight[k][1][i]) * xb;
          }
        }
        const float r = rsqrtf(team_sum(sum, w.team) * inv + s.eps);
        const float fall = r * r * (team_sum(dot, w.team) * inv);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const Lane<V, kNear> l(s, lane, k * w.team);
          float ya[V], yb[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float ua = x[j][k].a(i) * r, ub = x[j][k].b(i) * r;
            ya[i] = (na[k][i] * weight[k][0][i]) * r - ua * fall;
            yb[i] = (nb[k][i] * weight[k][1][i]) * r - ub * fall;
            // (an idle team has rotated a row of zeros by a token's angles, which may be NaN)
            grad[k][0][i] += on ? na[k][i] * ua : 0.f;
            grad[k][1][i] += on ? nb[k][i] * ub : 0.f;
          }
          Pairs<T, V, kNear> y;
          y.set(ya, yb);
          y.store(to + static_cast<int64_t>(h) * s.dim, l, on);
        }
        load(j, then, gthen, then_h + j * step, then_there);
      }
    }
  }
  if (partial == nullptr) return;
  // teams of a warp first, then the warps
  __shared__ float all[kThreads / 32][kMaxHeadDim];
  const int warp = threadIdx.x / 32;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Lane<V, kNear> l(s, lane, k * w.team);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = grad[k][m][i];
        for (int o = w.team; o < 32; o *= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        const int at = kNear ? l.at + 2 * i + m : (m ? l.at2 : l.at) + i;
        const bool has = kNear ? at < l.at + l.n + l.n2 : i < (m ? l.n2 : l.n);
        if (threadIdx.x % 32 < w.team && has) all[warp][at] = v;
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < s.dim; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kThreads / 32; ++u) v += all[u][i];
    partial[static_cast<int64_t>(blockIdx.x) * s.dim + i] = v;
  }
}

// 32 columns of one weight a block: its warps share the partial sums.
__global__ void __launch_bounds__(kThreads) heads_weights_kernel(const float* __restrict__ partial, int q_blocks, int k_blocks, int dim, void* dq, void* dk,
                                                                 bool f32, Elem type) {
  __shared__ float part[kThreads / 32][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, col = blockIdx.x * 32 + lane;
  const bool is_k = blockIdx.y != 0;
  void* to = is_k ? dk : dq;
  if (to == nullptr) return;
  const int blocks = is_k ? k_blocks : q_blocks;
  const float* from = partial + (is_k ? static_cast<int64_t>(q_blocks) * dim : 0) + col;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (col < dim) {
    int r = warp;
    for (; r + 24 < blocks; r += 32)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += from[static_cast<int64_t>(r + 8 * i) * dim];
    for (; r < blocks; r += 8) sum[0] += from[static_cast<int64_t>(r) * dim];
  }
  part[warp][lane] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  __syncthreads();
  if (warp == 0 && col < dim) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += part[i][lane];
    if (f32 || type == Elem::kF32) static_cast<float*>(to)[col] = v;
    else if (type == Elem::kF16) static_cast<__half*>(to)[col] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(to)[col] = __float2bfloat16_rn(v);
  }
}

// ---- choice of a form ---------------------------------------------------------------------------------------------
size_t size_of(Elem t) { return t == Elem::kF32 ? 4 : 2; }
bool fits(const HeadRows& r, const HeadsShape& s, int heads, size_t bytes) {
  if (r.data == nullptr) return true;
  const size_t e = size_of(s.type);
  return reinterpret_cast<uintptr_t>(r.data) % bytes == 0 && (s.batches <= 1 || r.batch * e % bytes == 0) &&
         (s.tokens <= 1 || r.token * e % bytes == 0) && (heads <= 1 || r.head * e % bytes == 0);
}
int pairs_of(const HeadsShape& s) { return s.rotary / 2 + (s.dim - s.rotary + 1) / 2; }
// Pairs a lane: 8, of fp32 4, where runs of so many divide both the rotated pairs and the others and every row is aligned to them
// (16 bytes); 4 of 16-bit types (8 bytes); else one.
int run_of(const HeadsShape& s, const Plan& w) {
  const size_t e = size_of(s.type);
  for (int run = e == 2 ? 8 : 4; run >= 4; run /= 2) {
    const size_t bytes = run * e;
    bool ok = s.rotary / 2 % run == 0 && (s.dim - s.rotary) % (2 * run) == 0 && reinterpret_cast<uintptr_t>(s.table) % 16 == 0;
    for (int i = 0; ok && i < w.sides; ++i) {
      const Side& d = w.side[i];
      ok = fits(d.x, s, d.heads, bytes) && fits(d.dy, s, d.heads, bytes) && reinterpret_cast<uintptr_t>(d.out) % bytes == 0 && d.out_token * e % bytes == 0;
    }
    if (ok) return run;
  }
  return 1;
}

constexpr int kFull = 512;  // threads of an SM that a launch should at least have
// A team takes as many of a token's heads as leave the device full of teams: what a token costs by itself, its place and its
// angles, is then spent once for many rows.  (As many teams to a token as a warp has, two rows each: 19 and 38 instructions a number
// forward and backward, where the arithmetic is 6 and 12.)
void cut(Plan& w, const HeadsShape& s, int run, int runs, int blocks_per_sm) {
  const int lanes = (pairs_of(s) + run - 1) / run;
  w.team = 1;
  while (w.team * runs < lanes) w.team *= 2;
  const int64_t tokens = s.batches * s.tokens, teams = kThreads / w.team;
  int heads = 0;
  for (int i = 0; i < w.sides; ++i) heads += w.side[i].heads;
  w.blocks = 0;
  for (int i = 0; i < w.sides; ++i) {
    Side& d = w.side[i];
    d.parts = 0;
    while ((1 << d.parts) < d.heads && (tokens << d.parts) * w.team < static_cast<int64_t>(kFull) * kSms * d.heads / heads) ++d.parts;
    d.units = tokens << d.parts;
    const int64_t most = std::max<int64_t>(1, static_cast<int64_t>(blocks_per_sm) * kSms * d.heads / heads);
    d.blocks = static_cast<int>(std::min((d.units + teams - 1) / teams, most));
    d.first = w.blocks;
    w.blocks += d.blocks;
  }
}
// One batch where the next one's tokens follow: no division in the kernels.
void flatten(HeadsShape& s, Plan& w) {
  if (s.batches <= 1) return;
  for (int i = 0; i < w.sides; ++i)
    for (const HeadRows* r : {&w.side[i].x, &w.side[i].dy})
      if (r->data != nullptr && r->batch != s.tokens * r->token) return;
  if (s.positions == nullptr || s.pos_batch != s.tokens * s.pos_token) return;
  s.tokens *= s.batches;
  s.batches = 1;
}
constexpr int kForwardBlocks = 16, kBackwardBlocks = 12;  // an SM, at most

template <typename T, int V, int K>
cudaError_t forward_run(const HeadsShape& h, Plan& w, cudaStream_t s) {
  cut(w, h, V, K, kForwardBlocks);
  constexpr int kRows = V == 1 || K > 1 ? 1 : 4;
  note_launch();
  if (h.interleaved) heads_forward_kernel<T, V, K, true, kRows><<<w.blocks, kThreads, 0, s>>>(h, w);
  else heads_forward_kernel<T, V, K, false, kRows><<<w.blocks, kThreads, 0, s>>>(h, w);
  return cudaGetLastError();
}
template <typename T>
cudaError_t forward_type(const HeadsShape& h, Plan& w, cudaStream_t s) {
  const int run = run_of(h, w);
  if constexpr (sizeof(T) == 2)
    if (run == 8) return forward_run<T, 8, 1>(h, w, s);
  if (run == 4) return pairs_of(h) <= 128 ? forward_run<T, 4, 1>(h, w, s) : forward_run<T, 4, 2>(h, w, s);
  return pairs_of(h) <= 64 ? forward_run<T, 1, 2>(h, w, s) : forward_run<T, 1, 8>(h, w, s);
}
template <typename T, int V, int K>
cudaError_t backward_run(const HeadsShape& h, Plan& w, float* partial, cudaStream_t s) {
  cut(w, h, V, K, kBackwardBlocks);
  constexpr int kRows = V == 1 || K > 1 ? 1 : 2;
  note_launch();
  if (h.interleaved) heads_backward_kernel<T, V, K, true, kRows><<<w.blocks, kThreads, 0, s>>>(h, w, partial);
  else heads_backward_kernel<T, V, K, false, kRows><<<w.blocks, kThreads, 0, s>>>(h, w, partial);
  return cudaGetLastError();
}
template <typename T>
cudaError_t backward_type(const HeadsShape& h, Plan& w, float* partial, cudaStream_t s) {
  const int run = run_of(h, w);
  if constexpr (sizeof(T) == 2)
    if (run == 8) return backward_run<T, 8, 1>(h, w, partial, s);
  if (run == 4) return pairs_of(h) <= 128 ? backward_run<T, 4, 1>(h, w, partial, s) : backward_run<T, 4, 2>(h, w, partial, s);
  return pairs_of(h) <= 64 ? backward_run<T, 1, 2>(h, w, partial, s) : backward_run<T, 1, 8>(h, w, partial, s);
}

bool shape_ok(const HeadsShape& s) {
  return s.dim > 0 && s.dim <= kMaxHeadDim && s.rotary >= 0 && s.rotary <= s.dim && s.rotary % 2 == 0 && s.heads > 0 && s.kv_heads > 0;
}

}  // namespace

cudaError_t launch_heads_forward(const HeadsForward& a, cudaStream_t s) {
  HeadsShape h = a.shape;
  if (!shape_ok(h)) return cudaErrorInvalidValue;
  if (h.batches * h.tokens == 0) return cudaSuccess;
  Plan w{};
  w.sides = 2;
  w.side[0] = {a.q, {}, static_cast<char*>(a.q_out), static_cast<int64_t>(h.heads) * h.dim, h.q_weight, h.heads};
  w.side[1] = {a.k, {}, static_cast<char*>(a.k_out), static_cast<int64_t>(h.kv_heads) * h.dim, h.k_weight, h.kv_heads};
  flatten(h, w);
  switch (h.type) {
    case Elem::kF32: return forward_type<float>(h, w, s);
    case Elem::kF16: return forward_type<__half>(h, w, s);
    default: return forward_type<__nv_bfloat16>(h, w, s);
  }
}

int heads_partials() { return kBackwardBlocks * kSms + 2; }

cudaError_t launch_heads_backward(const HeadsBackward& a, cudaStream_t s) {
  HeadsShape h = a.shape;
  if (!shape_ok(h)) return cudaErrorInvalidValue;
  if (h.batches * h.tokens == 0) return cudaSuccess;
  Plan w{};
  w.sides = a.dv_out != nullptr ? 3 : 2;
  w.side[0] = {a.q, a.dq, static_cast<char*>(a.dq_out), a.dq_token, h.q_weight, h.heads};
  w.side[1] = {a.k, a.dk, static_cast<char*>(a.dk_out), a.dk_token, h.k_weight, h.kv_heads};
  if (a.dv_out != nullptr) w.side[2] = {a.dv, {}, static_cast<char*>(a.dv_out), a.dv_token, nullptr, h.kv_heads};
  flatten(h, w);
  cudaError_t e;
  switch (h.type) {
    case Elem::kF32: e = backward_type<float>(h, w, a.partial, s); break;
    case Elem::kF16: e = backward_type<__half>(h, w, a.partial, s); break;
    default: e = backward_type<__nv_bfloat16>(h, w, a.partial, s);
  }
  if (e != cudaSuccess || a.partial == nullptr) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((h.dim + 31) / 32, 2);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  note_launch();
  return cudaLaunchKernelEx(&cfg, heads_weights_kernel, static_cast<const float*>(a.partial), w.side[0].blocks, w.side[1].blocks, h.dim, a.dq_weight,
                            a.dk_weight, h.weights_f32, h.type);
}

}  // namespace kern
}  // namespace mccl
