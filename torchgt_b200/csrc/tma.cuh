// Asynchronous copies of tiles from global into shared memory (TMA) and the barriers they complete on.
//
// Every map here is of a matrix of bf16 in rows of a multiple of 16 bytes; the x of every copy is a multiple of 64 values.  Loads past
// the matrix read zeros and count as whole.
#pragma once

#include <cuda.h>

#include "tensor_core.cuh"

namespace tgt {
namespace tma {

// Map of a [rows, columns] matrix of bf16, packed, for tiles of box_rows x 64 whose rows of 128 bytes lie in shared memory
// with the 128-byte swizzle.  TGT_ERR_CUDA with a message when the driver refuses.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int box_rows);

#ifdef __CUDACC__
__device__ __forceinline__ void prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void load(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void barrier_init(uint64_t* bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc::smem_address(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barriers_ready() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
// tc::wait by a whole warp, without the clock where the phase is complete or about to be: what feeds the tensor cores waits for
// every 64 of k.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t phase) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(tc::smem_address(bar)), "r"(phase) : "memory");
  return __all_sync(~0u, done != 0) || __all_sync(~0u, tc::wait(bar, phase));
}
// by its address, which may be another CTA's of the cluster
template <bool CLUSTER>
__device__ __forceinline__ void arrive(uint32_t bar) {
  if constexpr (CLUSTER) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expecting(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_address(bar)), "r"(bytes) : "memory");
}
#endif

}  // namespace tma
}  // namespace tgt
