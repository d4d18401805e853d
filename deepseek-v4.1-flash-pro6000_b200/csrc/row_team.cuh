// The CTAs of one cluster that share a logits row, a slice of its ids each ("team"): rank, barrier, and reads of another
// CTA's shared memory.  Such a read lies behind a team_barrier(), without which that CTA need not have started or written, and in
// front of another one (or of a team_arrive() whose team_wait() ends the kernel), without which it may have left.
#pragma once
#include <stdint.h>

namespace ds41 {

__device__ __forceinline__ uint32_t team_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t team_size() {
  uint32_t n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// All threads of all CTAs: what each has done before, to shared and to global memory, is seen by the others behind it.
__device__ __forceinline__ void team_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The barrier in two halves, with work in between that the others need not wait for.
__device__ __forceinline__ void team_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void team_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t team_address(const void *p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
  return a;
}
// CTA `rank`'s copy of a shared variable.
__device__ __forceinline__ uint32_t team_read(const uint32_t *p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(team_address(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 team_read(const float2 *p, uint32_t rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(team_address(p, rank)) : "memory");
  return v;
}

}  // namespace ds41
