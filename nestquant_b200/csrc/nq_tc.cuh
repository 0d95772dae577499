// What the kernels on the fifth-generation tensor cores share: mbarriers with bounded waits, tcgen05 fences, commits and tensor-memory stores, operand
// descriptors, the driver's tensor-map encoder.
#pragma once
#include <cuda.h>

#include "nq_common.cuh"

namespace nq {

constexpr long long kPfWaitNs = 2000000000ll;             // a wait that lasts 2 s is treated as a hang, unless the caller has another limit

// What the bounded waits of a CTA look at (shared memory).
struct PfWaits
{
    volatile int aborted;                // a wait has run out
    unsigned long long limit_ns;
};

__device__ __forceinline__ uint32_t saddr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(saddr(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive32(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) { mbar_arrive32(saddr(bar)); }
// The producer and MMA warps run their loops with all 32 lanes converged (so that addresses, descriptors and
// coordinates are warp-uniform values) and one elected lane issues the asynchronous instruction.
// Waits of a whole warp, `bar` a shared-space address.  What a wait costs that finds its phase complete is the branches around the
// poll, not the poll: 200 to 240 clocks as a loop (beside 16 busy warps), 95 as a poll, a vote and a branch that falls through, 15
// the poll alone.  So the poll that nearly always succeeds stands in line and the bounded loop behind a call.
// A wait returns false if it has run out, here or in another warp of the CTA.
__device__ __forceinline__ uint32_t mbar_poll(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
static __device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, PfWaits* waits)
{
    unsigned long long t0 = 0;
    for (;;)
    {
        if (__all_sync(0xffffffffu, mbar_poll(bar, parity))) return true;
        if (__any_sync(0xffffffffu, waits->aborted)) return false;
        unsigned long long t;            // (a poll that fails has waited for some time itself)
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t0 == 0) t0 = t;
        else if (__any_sync(0xffffffffu, t - t0 > waits->limit_ns)) break;
    }
    waits->aborted = 1;
    return false;
}
// Wait of a warp for what it has issued itself, whether or not the CTA has given up: no shared memory or tensor memory may be given back
// that a load or an MMA still touches.
static __device__ __noinline__ void mbar_wait_own(uint32_t bar, uint32_t parity)
{
    unsigned long long t0, t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
    do
    {
        if (__all_sync(0xffffffffu, mbar_poll(bar, parity))) return;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    } while (__all_sync(0xffffffffu, t - t0 < (unsigned long long)kPfWaitNs));
}
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, PfWaits* waits)
{
    if (__builtin_expect(__all_sync(0xffffffffu, mbar_poll(bar, parity)), 1)) return true;
    return mbar_wait_slow(bar, parity, waits);
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit_elect(uint64_t* bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(saddr(bar)) : "memory");
}
// 16 lanes x 4 x 256 bits of tensor memory from a warp, for columns 8 i .. 8 i + 7: lane (g, t4) supplies lane g columns
// 2 t4, 2 t4 + 1 (r[4 i], r[4 i + 1]) and lane g + 8, same columns (r[4 i + 2], r[4 i + 3]) - the layout of m16n8 fragments
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                   "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// shared-memory operand descriptor: start address, leading / stride byte offsets (all >> 4), descriptor version 1,
// layout 0 = no swizzle, 2 = 128-byte swizzle
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, uint32_t layout)
{
    const uint32_t lo = ((addr >> 4) & 0x3FFFu) | (((lbo >> 4) & 0x3FFFu) << 16);
    const uint32_t hi = ((sbo >> 4) & 0x3FFFu) | (1u << 14) | (layout << 29);
    return ((uint64_t)hi << 32) | lo;
}
// A value that is the same in all lanes, as one that the compiler knows to be: what it cannot tell from a lane's own value (anything
// loaded, anything that depends on the thread index) reaches the uniform registers of an MMA or TMA instruction by a move of its own
// in front of every one.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled()
{
    static EncodeTiledFn fn = nullptr;
    if (!fn)
    {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || !p) return nullptr;
        fn = (EncodeTiledFn)p;
    }
    return fn;
}

}  // namespace nq
