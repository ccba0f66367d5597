// Asynchronous copies of tiles between global and shared memory (TMA) and the barriers they complete on.
//
// Every map here is of a matrix of bf16 in rows of a multiple of 16 bytes; the x of every copy is a multiple of 32 values.  Loads past
// the matrix read zeros and count as whole, stores past it are dropped.
#pragma once

#include <cuda.h>

#include "tensor_core.cuh"

namespace tgt {
namespace tma {

// Map of a [rows, columns] matrix of bf16, packed, for tiles of box_rows x box_columns whose rows, 64 or 128 bytes, lie in
// shared memory with that swizzle.  TGT_ERR_CUDA with a message when the driver refuses.
int make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t columns, int box_rows, int box_columns);

#ifdef __CUDACC__
__device__ __forceinline__ void prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void load(uint32_t to, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
      "l"(map), "r"(x), "r"(y), "r"(tc::smem_address(bar))
      : "memory");
}
__device__ __forceinline__ void store(const CUtensorMap* map, uint32_t from, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(from), "r"(x),
               "r"(y)
               : "memory");
}
// One thread's stores: a group of them; until all but the last PENDING groups have been read from shared memory; until all
// have been written.
__device__ __forceinline__ void end_group() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void groups_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory"); }
__device__ __forceinline__ void groups_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void barrier_init(uint64_t* bar, int arrivals) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tc::smem_address(bar)), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void barriers_ready() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_address(bar)) : "memory");
}
__device__ __forceinline__ void arrive_expecting(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_address(bar)), "r"(bytes) : "memory");
}
#endif

}  // namespace tma
}  // namespace tgt
