// Launchers of the 8-bit activation checkpoints (plain C++ header).
#pragma once

#include <cuda_runtime_api.h>

#include <cstdint>

namespace mccl {
namespace kern {

enum class Elem { kF32, kF16, kBF16 };

// Groups of 64 numbers of a row share a scale: `scales` [rows, groups].  `codes`: rows of `pitch` bytes, a multiple of 16 that
// holds the row; what is beyond the row is zero.
struct Packed8Rows {
  int8_t* codes;
  float* scales;
  int64_t rows, cols, pitch;
};
inline int64_t pack8_groups(int64_t cols) { return (cols + 63) / 64; }
inline int64_t pack8_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }

// x: rows of `ld` elements.
cudaError_t launch_pack8(const void* x, Elem type, int64_t ld, const Packed8Rows& p, cudaStream_t s);
cudaError_t launch_unpack8(const Packed8Rows& p, void* x, Elem type, int64_t ld, cudaStream_t s);

}  // namespace kern
}  // namespace mccl
