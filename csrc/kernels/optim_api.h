// Launcher of the fused multi-tensor AdamW kernel (plain C++ header).
#pragma once

#include <cuda_runtime_api.h>
#include <vector_types.h>

#include <cstdint>

namespace mccl {
namespace kern {

// Elements handled by one CTA: 256 threads, four 16-byte vectors of each array, two of them in flight together.
// (Chunks of 16384 with one vector in flight: 85 M parameters 385 us, 6.17 TB/s; so: 362 us, 6.56 TB/s, and a
// small model spreads over four times as many SMs.)
constexpr int kAdamWChunk = 4096;

// All pointers are device pointers; arrays are indexed by tensor id.
struct AdamWTable {
  const uint64_t* params;      // float* per tensor
  const uint64_t* grads;       // const float* per tensor
  const uint64_t* exp_avg;     // float* per tensor
  const uint64_t* exp_avg_sq;  // float* per tensor
  const int64_t* sizes;        // elements per tensor
  const int2* chunks;          // per CTA: {tensor id, chunk index}
  int num_chunks;
};

struct AdamWHyper {
  float lr;
  float beta1, beta2;
  float eps;
  float weight_decay;
  float step_size;       // lr / (1 - beta1^t)
  float inv_sqrt_bias2;  // 1 / sqrt(1 - beta2^t)
  float grad_scale;      // multiplied into every gradient first
};

// `max_ctas` > 0 caps the grid (each CTA then walks several chunks): a step that runs beside other
// kernels (a bucket's update during backward) can be kept to a share of the SMs and of HBM bandwidth.
cudaError_t launch_adamw_multi(const AdamWTable& tab, const AdamWHyper& h, cudaStream_t s, int max_ctas = 0);

// ---- tensors of several kinds (kernels/adamw_kinds.cu) ---------------------------------------------
// Moments that share one scale where they are kept in 8 bits.
constexpr int kMomentGroup = 256;
// Numbers of a CTA: with few, more CTAs share a small step; with many, each starts less often.  us by 2048 and by 8192: 1 M numbers 16 and 22, 12 M 50
// and 51, 24 M 85 and 84, 96 M 290 and 269 (bf16 parameters: 16 and 24, 46 and 51, 80 and 81, 269 and 271); fp32 moments, of which fewer are on
// their way, 16 and 20, 62 and 69, 110 and 119, 396 and 411.
inline int adamw_kinds_chunk(int64_t numbers, bool eight) { return eight && numbers >= 24ll << 20 ? 8192 : 2048; }

// One tensor, in device memory.
struct AdamWTensor {
  void* param;              // fp32 or, `half`, bf16
  void* exp_avg;            // fp32 or, `eight`, e4m3 padded to whole groups
  void* exp_avg_sq;         // fp32 or e5m2, alike
  float* exp_avg_scale;     // of each group
  float* exp_avg_sq_scale;
  int16_t* low;             // what a bf16 parameter leaves of its fp32 value's bits
  int64_t size;
  int32_t half, eight, aligned, unused;  // aligned: all but the gradient begin at multiples of 16 bytes
};
// The hyper-parameters of one step, each rounded from 64 bits once.
struct AdamWStep {
  float beta1, one_less_beta1, beta2, one_less_beta2, eps;
  float decay;           // 1 - lr wd
  float step_size;       // lr / (1 - beta1^t)
  float inv_sqrt_bias2;  // 1 / sqrt(1 - beta2^t)
  float grad_scale;
  float one;             // 1
  uint32_t ordinary;     // eps and inv_sqrt_bias2 are far from either end of fp32's range
  uint32_t step_word;    // t times the golden ratio's digits, for the dither
  int chunk;             // numbers of a CTA, whole groups
};
cudaError_t launch_adamw_kinds(const AdamWTensor* tensors, const uint64_t* grads, const int2* chunks, int num_chunks, const AdamWStep& h, cudaStream_t s,
                               int max_ctas = 0);
// For tests: the step's root of each b and its quotients a / b.
cudaError_t launch_root_quotient(const float* a, const float* b, float* root, float* quotient, int64_t n, cudaStream_t s);

}  // namespace kern
}  // namespace mccl
