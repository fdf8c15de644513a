// The CTAs of a thread-block cluster and their shared memory.
#pragma once

#include "common.cuh"

namespace fo {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// As cluster_barrier, but orders no memory: does not wait for stores on their way.
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ uint32_t remote_address(const void* p, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(shared_address(p)), "r"(cta));
  return r;
}
// A float into CTA `cta`'s copy of `to`; seen there behind a cluster_barrier.
__device__ __forceinline__ void store_remote(float* to, uint32_t cta, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote_address(to, cta)), "f"(v) : "memory");
}

}  // namespace fo
