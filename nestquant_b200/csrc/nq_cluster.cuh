// CTAs of a cluster: barrier and distributed shared memory.
#pragma once
#include <stdint.h>

namespace nq {

// every thread of every CTA of the cluster arrives and waits
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_address(uint32_t address, int rank)
{
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
    return there;
}
__device__ __forceinline__ void cluster_store(uint32_t address, float x, float y)
{
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" :: "r"(address), "f"(x), "f"(y) : "memory");
}

}  // namespace nq
