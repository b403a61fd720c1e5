// Launchers of the gated feed-forward block's products (plain C++ header), and of a linear layer's, which are of the same kind.
//
//     g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//
// of `tokens` rows, `width` numbers in and out, `hidden` between.  Six products; what stands between them is inside of them.
//
//     y = act(x W^T + b) + r
//
// of `tokens` rows, `hidden` numbers in and `width` out: its product is kDown's with what follows it, and its gradients are kBack and kWeightDown.
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

#include "kernels/pack8_api.h"

namespace mccl {
namespace kern {

enum class GatedProduct {
  kUp,          // a0 = x, b0 = Wg, b1 = Wu: h to out0, g and u to `kept`
  kDown,        // a0 = h, b0 = Wd: y to out0
  kGate,        // a0 = dy, b0 = Wd: with dh = dy Wd: h to out0, dg to out1, du to out2, from `kept`
  kInput,       // a0 = dg, a1 = du, b0 = Wg, b1 = Wu: dx to out0
  kWeightUp,    // a0 = dg, a1 = du, b0 = x: dWg to out0, dWu to out1
  kWeightDown,  // a0 = dy, b0 = h: dWd to out0
  kLayer,       // a0 = x, b0 = W: y to out0, x W^T + b to out1 (rows of gated_row(width)) where it is kept
  kBack,        // a0 = dz, b0 = W: dx to out0
};
enum class GatedActivation { kSilu, kGeluTanh };
// How g and u wait for the backward pass: not at all, as floats of three bytes, as codes of 8 bits.
enum class GatedKeep { kNone, kWide, kEight };

struct GatedShape {
  int64_t tokens, width, hidden;
  bool bf16;  // else fp16
  GatedActivation activation;
  GatedKeep keep;
};
// Elements from row to row of h, dg and du: `hidden` padded to whole groups; what is beyond `hidden` is zero.
inline int64_t gated_pitch(int64_t hidden) { return (hidden + 63) / 64 * 64; }
int64_t gated_kept_bytes(const GatedShape& s);

// Rows of 16-bit numbers, 16-byte aligned and so many elements apart.
struct GatedOperand {
  const void* data;
  int64_t ld;
};
struct GatedArgs {
  GatedProduct product;
  GatedOperand a0, a1, b0, b1;
  void *out0, *out1, *out2;
  int64_t ldo;          // of the outputs; of h, dg and du gated_pitch
};
// What follows the product of a linear layer.
enum class LayerActivation { kNone, kRelu, kSilu, kGelu, kGeluTanh };
struct LayerFinish {
  LayerActivation activation;
  const void* bias;      // `width` numbers of the operands' type, or null
  const void* residual;  // rows of y's type, `ldr` numbers apart, or null
  int64_t ldr;
  bool y_f32;            // else of the operands' type
};
struct GatedLaunch {
  GatedShape shape;
  const LayerFinish* layer;  // of kLayer, or null
  void* kept;
  float* partial;       // gated_partial_bytes
  uint32_t* failed;     // set to 1 where a wait runs out, whose tiles then are NaN; or null
  int64_t wait_limit;   // cycles of a quarter of a wait; negative: about a second in all
};
// One product, or up to three of kDown, kInput, kWeightUp, kWeightDown and kBack: side by side where that is faster.
int64_t gated_partial_bytes(const GatedProduct* p, int n, const GatedShape& s);
cudaError_t launch_gated(const GatedArgs* g, int n, const GatedLaunch& r, cudaStream_t s);

// Matrices of 16-bit numbers whose rows are not 16-byte aligned (or whose numbers do not lie side by side) copied to ones that are,
// up to five in one launch.  `beside`: without waiting for the last launch_gated before it on this stream, nor for anything launched
// behind that one; neither it nor these may read or write `to` or write `from`.  So `to` was allocated before that launch, at which all
// earlier work on the stream is done: a block that the allocator hands out later may have been another thread's, whose kernels still run.
struct GatedCopy {
  const void* from;
  int64_t row_stride, col_stride, rows, cols;  // elements
  void* to;                                    // 16-byte aligned
  int64_t ld;                                  // gated_row(cols)
};
inline int64_t gated_row(int64_t cols) { return (cols + 7) / 8 * 8; }
constexpr int kGatedCopies = 5;
cudaError_t launch_gated_copies(const GatedCopy* jobs, int n, bool beside, cudaStream_t s);

// A whole forward pass of few rows, two launches that read the weights at the rate of memory (kernels/gated_few.cu).  Rows of any
// alignment.  `h`: scratch of tokens x gated_pitch(hidden) x 4 bytes.
constexpr int64_t kFewTokens = 32;
// Whether it is faster than the tiles, whose matrix instructions cost the same for any number of tokens and whose launches cost more.
// By the weights' size alone, which near the limits is as often a little wrong as right: for 2 tokens the kernels here gain 9 us of 4096 x
// 10240 and lose 5 of 5120 x 8192, just as many numbers.
// us, here and by tiles: 2 tokens 4096 x 10240 59 and 68, 5120 x 8192 64 and 59, 5120 x 13824 98 and 93; 8 tokens 4096 x 6144 40 and 44,
// 5120 x 8192 70 and 59; 16 tokens 2048 x 4096 25 and 26, 2048 x 5632 32 and 30; 32 tokens 1024 x 2816 18 and 19, 1536 x 4096 27 and 25.
inline bool gated_is_few(const GatedShape& s) {
  const int64_t n = s.width * s.hidden;
  return n <= (s.tokens <= 2 ? 48 << 20 : s.tokens <= 8 ? 32 << 20 : s.tokens <= 16 ? 8 << 20 : s.tokens <= kFewTokens ? 4 << 20 : 0);
}
// fp32, against three products of the linear layer and the gate between them, us: 8 tokens 256 x 704 7 and 15, 1024 x 2816 20 and 40, 1481 x
// 4108 53 and 55, 4096 x 10240 148 and 234; 16 tokens 10 and 23, 34 and 41, 93 and 56, 251 and 256.  (The host's part: 12 and 31.)
inline bool gated_is_few_f32(const GatedShape& s) { return s.tokens <= 8 || (s.tokens <= 16 && s.width * s.hidden <= (4 << 20)); }
struct GatedFew {
  GatedShape shape;
  GatedOperand x, w_gate, w_up, w_down;
  void* h;
  void* y;   // rows of `width`
  bool f32;  // all of them, whatever `shape` says
};
cudaError_t launch_gated_few(const GatedFew& g, cudaStream_t s);

// The same in fp32, between products of their own (kernels/gate_f32.cu): rows of g and u, `ld` numbers apart, to rows of h; rows of
// g with u behind them and dh to rows of dg with du behind them.
cudaError_t launch_gate_f32(const float* g, const float* u, int64_t ld, float* h, int64_t rows, int64_t cols, GatedActivation act, cudaStream_t s);
cudaError_t launch_gate_f32_backward(const float* gu, const float* dh, float* dgu, int64_t rows, int64_t cols, GatedActivation act, cudaStream_t s);

// ---- linear layer -------------------------------------------------------------------------------------------
// A layer of few rows, one launch that reads the weights at the rate of memory (kernels/linear_few.cu).  Rows of any alignment, which the tiles would
// have copied.
// us of bf16 from memory, here and by tiles (of which a narrow layer has few, each with all of the reduction): 1 token 1024 x 1024 2.5 and 5.1, 1024 x 4096
// 6.1 and 5.8, 4096 x 4096 11.4 and 14.2, 2048 x 8192 12 and 9.5, 4096 x 10240 26 and 20; 16 tokens 2048 x 2048 5.5 and 8.4, 8192 x 2048 16 and 25, 4096 x
// 4096 16.3 and 14.2; rows that begin anywhere, 1723 x 5258, 1 token 16 and 22, 16 tokens 21 and 22, 32 tokens 32 and 23.
inline bool layer_is_few(int64_t tokens, int64_t out, bool aligned) {
  return tokens <= 8 ? out <= 4096 || !aligned : tokens <= 16 ? out <= 2560 || !aligned : tokens <= kFewTokens && out <= 2560;
}
struct LayerFew {
  int64_t tokens, in, out;
  bool bf16;  // else fp16
  GatedOperand x, weight;
  LayerFinish finish;
  void* y;  // rows of `out`
};
cudaError_t launch_layer_few(const LayerFew& g, cudaStream_t s);

// A layer of some tens or hundreds of rows, on smaller tiles (kernels/linear_tiles.cu).  layer_tile: their columns, or 0 where they would be more than
// one for each SM and launch_gated's kLayer takes the product.
int layer_tile(int64_t tokens, int64_t in, int64_t out);
struct LayerTiles {
  int64_t tokens, in, out;
  bool bf16;  // else fp16
  GatedOperand x, weight;  // aligned to 16 bytes
  LayerFinish finish;
  void *y, *z;            // as kLayer's
  uint32_t* failed;
  int64_t wait_limit;
};
cudaError_t launch_layer_tiles(const LayerTiles& g, cudaStream_t s);

// A small layer of fp32, each direction one launch (kernels/linear_small.cu, with both sides measured): short reductions, and so little to multiply that
// products of the library and passes around them are mostly their launches.  What is gained is the host's time, 6 to 10 us a call forward and 33 with gradients:
// on the device a few shapes are slower by it than by the library (3 x 256 x 192 6.5 us for 2.7, 1024 x 256 x 256 11.4 for 9.8), which shows where calls are
// replayed from a graph or wait behind longer ones.
inline bool layer_is_small(int64_t tokens, int64_t in, int64_t out) { return in <= 256 && tokens <= 8192 && out <= 8192 && tokens * in * out <= 1ll << 26; }
inline bool layer_is_small_backward(int64_t tokens, int64_t in, int64_t out) {
  return out <= 512 && tokens <= 1024 && in <= 8192 && tokens * in * out <= 1ll << 26;
}
struct LayerSmall {
  int64_t tokens, in, out;
  const float *x, *weight, *bias, *residual;  // rows ld.. apart; bias and residual may be null
  int64_t ldx, ldw, ldr;
  LayerActivation activation;
  float *y, *z;  // rows of `out`; z null where it is not kept
};
cudaError_t launch_layer_small(const LayerSmall& g, cudaStream_t s);
struct LayerSmallBackward {
  int64_t tokens, in, out;
  const float *dz, *x, *weight;
  int64_t ldz, ldx, ldw;
  float *dx, *dw, *dbias;  // one behind the other; null where nobody asks
};
cudaError_t launch_layer_small_backward(const LayerSmallBackward& g, cudaStream_t s);

// What stands around the products, in one pass each (kernels/linear_pass.cu).  Rows `ld` numbers apart of one type.
struct LayerRows {
  const void* data;
  int64_t ld;
  Elem type;
};
// y = act(z) + residual, of fp32 rows one behind the other (`residual.data` null without one).
cudaError_t launch_layer_finish(const float* z, const LayerRows& residual, float* y, int64_t rows, int64_t cols, LayerActivation act, cudaStream_t s);
// dz = dy act'(z) to rows of `dz_ld` numbers (null: only the sums), and the sums of dy act'(z) over the rows, before it is rounded, to `bias`
// (null: none), in a fixed order.  `z.data` null: dz = dy.
struct LayerDerive {
  int64_t rows, cols;
  LayerRows dy, z;
  LayerActivation activation;
  void* dz;
  int64_t dz_ld;
  Elem dz_type;
  void* bias;
  Elem bias_type;
  float* partial;  // layer_partial_bytes
};
int64_t layer_partial_bytes(int64_t rows, int64_t cols);
cudaError_t launch_layer_derive(const LayerDerive& g, cudaStream_t s);

}  // namespace kern
}  // namespace mccl
