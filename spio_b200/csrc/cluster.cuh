// Barriers of a thread-block cluster and loads from the shared memory of its CTAs.
#pragma once

#include "ptx.cuh"

namespace spio_b200 {

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
// For threads that have neither written what another CTA reads nor read another CTA's memory: it orders nothing, so that
// loads issued before it may still be under way when the other CTAs pass the barrier and leave.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// *p of the CTA `rank` of the cluster
__device__ __forceinline__ float2 cluster_load(const float2* p, int rank) {
  u32 at;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float cluster_load(const float* p, int rank) {
  u32 at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

}  // namespace spio_b200
