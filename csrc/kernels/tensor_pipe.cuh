// What kernels on the fifth-generation tensor cores share: barriers with bounded waits, boxes by TMA, matrix descriptors, tensor memory, tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kernels/gated_api.h"

namespace mccl {
namespace kern {
namespace {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
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
// Into this CTA's own shared memory, for this CTA alone.
__device__ __forceinline__ void load_own_box(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x),
               "r"(y), "r"(bar)
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

// ---- host ---------------------------------------------------------------------------------------------------
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
  while (n < rows && n < 128) n *= 2;
  return n;
}
bool make_map(CUtensorMap* map, const GatedOperand& m, int64_t inner, int64_t outer, uint32_t box_rows, bool bf16, bool f32 = false) {
  const int64_t size = f32 ? 4 : 2;
  if (m.data == nullptr || reinterpret_cast<uintptr_t>(m.data) % 16 != 0 || m.ld * size % 16 != 0 || m.ld < inner || inner > 0x7FFFFFFF || outer > 0x7FFFFFFF) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)}, strides[1] = {static_cast<cuuint64_t>(m.ld * size)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), box_rows}, one[2] = {1, 1};
  return encode_tiled()(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(m.data), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace kern
}  // namespace mccl
