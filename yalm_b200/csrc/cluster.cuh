// Thread-block clusters: ranks, the barrier, and addresses in another CTA's shared memory.
#pragma once

#include <stdint.h>

namespace yb {

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// Every thread of every CTA of the cluster arrives (release: its shared-memory writes become
// visible to the other CTAs) and waits for all others (acquire).
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The same in two parts: a CTA that has arrived may go on with what the others do not read.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// Generic address of the same shared-memory variable in CTA `rank` of the cluster (distributed
// shared memory): plain loads through it, which the compiler may batch, read the peer's copy.
template <typename T>
__device__ __forceinline__ const T* dsmem_ptr(const T* local, uint32_t rank) {
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(local), "r"(rank));
  return reinterpret_cast<const T*>(r);
}

}  // namespace yb
