// Launchers of layer norm, with the sum before it, and its gradients (plain C++ header).
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

#include "kernels/pack8_api.h"

namespace mccl {
namespace kern {

// Rows of numbers of one type, `ld` of them from one to the next; null where there are none.
struct NormRows {
  const void* data;
  int64_t ld;
  Elem type;
};
constexpr int64_t kNormMostCols = 0x7FFF0000;
struct NormShape {
  int64_t rows;
  int cols;
  float eps;
  const void *weight, *bias;  // `cols` numbers of one type, or null
  Elem weight_type;
};
// s = x + residual, kept in the residual's type (without one s is x); y = (s - mean) rstd weight + bias.
struct NormForward {
  NormShape shape;
  NormRows x, residual;
  void* sum;           // rows of `cols` numbers of the residual's type; null without one
  void* y;             // rows of `cols` numbers
  Elem y_type;
  float *mean, *rstd;  // of each row, or null
};
// dx = rstd (g - mean(g) - u mean(g u)) + ds with g = dy weight, u = (s - mean) rstd; dweight = sum of dy u, dbias = sum of dy.
struct NormBackward {
  NormShape shape;
  NormRows s, dy, ds;          // ds: null, or of the type of s
  const float *mean, *rstd;
  void *dx, *dresidual;        // rows of `cols` numbers; null where nobody asks, or where the two are the same
  Elem dx_type;                // dresidual's is that of s
  void *dweight, *dbias;       // of the weight's type; null where nobody asks
  float* partial;              // norm_partial_bytes
};
cudaError_t launch_norm_forward(const NormForward& a, cudaStream_t s);
int64_t norm_partial_bytes(const NormShape& s);
cudaError_t launch_norm_backward(const NormBackward& a, cudaStream_t s);

}  // namespace kern
}  // namespace mccl
