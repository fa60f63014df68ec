// Sums over the CTAs of a cluster through distributed shared memory: each CTA leaves its partial tile at the
// same place of its own shared memory, each adds up its share of the outputs from all of them.
#pragma once

#include <stdint.h>

namespace cogni {
namespace {

__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void split_sync() {  // all threads of all CTAs of the cluster
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The sum over the parts of four consecutive tile rows, in the order of the parts.
__device__ __forceinline__ float4 sum_parts(uint32_t own, int splits) {
  float4 a = ld_peer4(peer_smem(own, 0));
  for (int z = 1; z < splits; z++) {
    const float4 b = ld_peer4(peer_smem(own, z));
    a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
  }
  return a;
}

}  // namespace
}  // namespace cogni
