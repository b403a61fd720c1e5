// Launchers of the norms and the rotation of queries and keys (plain C++ header).
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

#include "kernels/pack8_api.h"

namespace mccl {
namespace kern {

// Rows of `dim` elements, one for each head of each token; strides in elements.
struct HeadRows {
  const void* data;
  int64_t batch, token, head;
};
// What both directions are told.  Table: [positions, 2, rotary / 2], cosines and then sines; a position outside of it rotates
// by NaN.
struct HeadsShape {
  int64_t batches, tokens;
  int heads, kv_heads, dim, rotary;
  bool interleaved;
  float eps;
  Elem type;
  const void *q_weight, *k_weight;
  bool weights_f32;   // else of `type`
  const float* table;
  int64_t table_rows;
  const void* positions;   // int32 or int64; null: 0, 1, ... in each batch
  bool positions_32;
  int64_t pos_batch, pos_token;   // strides
};
constexpr int kMaxHeadDim = 512;

// q_out [batches, tokens, heads, dim], k_out likewise.
struct HeadsForward {
  HeadsShape shape;
  HeadRows q, k;
  void *q_out, *k_out;
};
cudaError_t launch_heads_forward(const HeadsForward& a, cudaStream_t s);

// Gradients to rows that are `dx_token` elements a token apart from each other: queries from dq_out on, keys from dk_out on, and
// where dv_out is not null the rows of dv copied there.
struct HeadsBackward {
  HeadsShape shape;
  HeadRows q, k, dq, dk, dv;
  void *dq_out, *dk_out, *dv_out;
  int64_t dq_token, dk_token, dv_token;
  float* partial;                // heads_partials() x dim, or null: no gradients of the weights
  void *dq_weight, *dk_weight;   // of the weights' type; or null
};
int heads_partials();
cudaError_t launch_heads_backward(const HeadsBackward& a, cudaStream_t s);

}  // namespace kern
}  // namespace mccl
