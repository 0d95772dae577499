// Products with 4-bit weights (nq_w4.cuh) for calls of many rows: on the fifth-generation tensor cores, 128 rows of the matrix times TOKENS rows of x per item.
//
//   sums       (8 warps) a warp has 32 rows of the matrix (its quarter of tensor memory) and half of the tokens; adds every
//              group's sums, times the group's scale, to its registers, and writes the item's results
//   weights    (8 warps for 128 tokens, else 16) a warp streams one strip of 16 rows, or every other chunk of it (W4Stream), turns a unit into exact
//              halves q - z and stores them as the MMA's A operand in tensor memory (16x256b stores take the fragments as they are)
//   TMA        (one warp) the tokens' tiles [TOKENS x 64], two per chunk of 128 columns
//   MMAs       (one warp) an elected lane issues tcgen05.mma, 128 x TOKENS x 16 a step, into one of two accumulators per group of columns: an accumulator
//              holds one group's sum only, so that the scale is applied in 32 bits and nothing is rounded before the result
// Bound by the tensor pipe by intent; in practice at 128 rows an item by the sums, which read 128 x 128 of tensor memory a chunk, and the MMAs, which wait for
// one another over two accumulators: a chunk takes 820 clocks, 512 of them MMAs; weights are three chunks ahead.  us, rows of 4,096 x 6,144 in groups of 128 (tensor
// floor): 32 9.4, 64 11.0, 128 13.4 (3.9), 256 18.0 (7.8), 512 24.3 (15.7), 2,048 95 (62.8) = 1.08 PFLOP/s; 512 rows in groups of 64 35, of 32 55: two and four times the
// sums.  What made the difference at 512 rows: one row block of 32 per pass of the other kernel 156; this kernel with eight warps of 128 tokens' sums and the MMAs one by
// one 35; registers by role and two sums an instruction 30; one vote for a chunk's three barriers 24.6.  In groups of 64: scales that stay where they were loaded and
// the next barrier looked at behind the products 36.5 -> 33.5; in groups of 32: an accumulator read at once 58 -> 55.  Passes of up to 64 rows: an MMA of 16 columns takes
// ~56 clocks however few tokens it has, and sixteen warps decode.  Passes of 64 rows in groups of 64 and 32 spill: 832 threads have 72 registers each, and the sums
// want more, 16 to 32 bytes with fp16 scales, 194 to 244 with bf16 ones; 64 rows of 4,096 x 6,144 take 11.9 and 14.7, with bf16 scales 14.1 and 17.5 (groups of 128, which
// do not spill: 10.8 and 11.2).
// Columns of an item may be split over a cluster; each CTA then adds up a share of the tokens, the others' sums come through distributed shared memory.
// Every mbarrier wait is bounded (nq_tc.cuh): on time-out the CTA raises status[0], waits for its loads and MMAs in flight and ends.
#include <stddef.h>

#include "nq_tc.cuh"
#include "nq_w4.cuh"

namespace nq {

struct WgShared {
    uint64_t full_a[6], full_b[6], empty[6], sum_full[2], sum_empty[2], done;
    uint32_t tmem;
    PfWaits waits;
    int row[kW4MaxExperts + 1], first[kW4MaxExperts + 2], warp_sums[32];
};
template <int GROUPS, int TOKENS>
struct WgPlan {
    static constexpr int kSumWarps = 8, kDecodeWarps = TOKENS == 128 ? 8 : 16, kHalves = kDecodeWarps / 8;      // (kHalves warps to a strip)
    static constexpr int kTma = kSumWarps + kDecodeWarps, kMma = kTma + 1;                                      // the other two warps
    static constexpr bool kSplit = TOKENS == 128;                         // registers go by warpgroup: 144 for sums, 72 for weights, 48 for the rest, of 5 x 96
    static constexpr int kThreads = kSplit ? 640 : 32 * 26;
    static constexpr int kColumns = TOKENS / 2;                           // tokens of a sum warp
    using Stream = W4Stream<GROUPS, 4, kHalves>;
    // groups whose sums are kept side by side in one of the two accumulators: the waits are per accumulator
    static constexpr int kSet = GROUPS * TOKENS <= 128 ? GROUPS : 128 / TOKENS, kSumColumns = kSet * TOKENS;
    static constexpr int kStages = kSumColumns == 128 ? 4 : 6;                 // chunks ahead; a weight tile is 64 columns of tensor memory
    static constexpr int kBox = TOKENS * 128;                             // a token tile of 64 columns
    static constexpr int kTiles = kStages * 2 * kBox, kPlanes = kDecodeWarps * Stream::kBytes, kSums = TOKENS * 512;
    // tiles, and after them, or in their place once they are through, the sums of a split item; planes
    static constexpr int kRest = kTiles > kSums ? kTiles : kSums, kSmem = kRest + kPlanes + (int)sizeof(WgShared);
    static_assert(kSmem <= 232448, "shared memory of a CTA");
};

extern __shared__ __align__(1024) uint8_t wg_smem[];

__device__ __forceinline__ void tma_two_boxes(uint32_t dst, uint32_t box, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(2 * box) : "memory");
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst + box), "l"(map), "r"(x + 64), "r"(y), "r"(bar) : "memory");
}
// The MMAs of a group of STEPS steps of 16 columns, by one elected lane (one election, few instructions: this warp shares its scheduler with busy ones), with FULL the
// commit to the barrier `full` and with EMPTY that to `empty`.  Weights in tensor memory, 8 columns a step; tokens in shared memory, two tiles of 64 columns, BOX bytes
// apart (the descriptor counts in 16 bytes).  The first MMA overwrites the accumulator.
#define NQ_WG_STEP(A, B, P) \
    "add.u32 ta, %1, " A ";\n\tadd.u32 tb, %2, " B ";\n\tmov.b64 db, {tb, %3};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [ta], db, %4, " P ";\n\t"
#define NQ_WG_COMMIT(BAR) "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [" BAR "];\n\t"
#define NQ_WG_GROUP(STEPS_TEXT, COMMITS)                                                                                                                      \
    asm volatile("{\n\t.reg .pred p, q, e;\n\t.reg .b64 db;\n\t.reg .b32 ta, tb;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %4, %4;\n\tsetp.eq.u32 q, %4, %4;\n\t"  \
                 STEPS_TEXT COMMITS "}"                                                                                                                \
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(full), "n"(BOX >> 4), "r"(empty) : "memory")
#define NQ_WG_EITHER(STEPS_TEXT)                                                             \
    do {                                                                                     \
        if (FULL && EMPTY) NQ_WG_GROUP(STEPS_TEXT, NQ_WG_COMMIT("%5") NQ_WG_COMMIT("%7"));   \
        else if (FULL) NQ_WG_GROUP(STEPS_TEXT, NQ_WG_COMMIT("%5"));                          \
        else NQ_WG_GROUP(STEPS_TEXT, "");                                                    \
    } while (0)
template <int STEPS, int BOX, bool FULL, bool EMPTY>
__device__ __forceinline__ void mma_group(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t full, uint32_t empty)
{
    static_assert(FULL || !EMPTY, "a chunk's last group is the last of an accumulator");
    if constexpr (STEPS == 8)
        NQ_WG_EITHER(NQ_WG_STEP("0", "0", "p") NQ_WG_STEP("8", "2", "q") NQ_WG_STEP("16", "4", "q") NQ_WG_STEP("24", "6", "q")
                     NQ_WG_STEP("32", "%6", "q") NQ_WG_STEP("40", "%6+2", "q") NQ_WG_STEP("48", "%6+4", "q") NQ_WG_STEP("56", "%6+6", "q"));
    else if constexpr (STEPS == 4)
        NQ_WG_EITHER(NQ_WG_STEP("0", "0", "p") NQ_WG_STEP("8", "2", "q") NQ_WG_STEP("16", "4", "q") NQ_WG_STEP("24", "6", "q"));
    else
        NQ_WG_EITHER(NQ_WG_STEP("0", "0", "p") NQ_WG_STEP("8", "2", "q"));
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr) : "memory");
}
// (the registers pass through the wait: nothing reads them in front of it)
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                   "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]) :: "memory");
}

// two 32-bit floats in a register pair
__device__ __forceinline__ uint64_t two_floats(float v) { return (uint64_t)__float_as_uint(v) << 32 | __float_as_uint(v); }
__device__ __forceinline__ float one_of(uint64_t v, int i) { return __uint_as_float((uint32_t)(i ? v >> 32 : v)); }
// sum += s * (x, y)
__device__ __forceinline__ void fma_two(uint64_t& sum, uint64_t s, uint32_t x, uint32_t y)
{
    asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%2, %3};\n\tfma.rn.f32x2 %0, %1, v, %0;\n\t}" : "+l"(sum) : "l"(s), "r"(x), "r"(y));
}

// mbar_poll that does not wait
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// (mbar_wait_warp with its slow part in line: a call would take the registers that the sums are in)
__device__ __forceinline__ bool wait_bar_slow(uint32_t bar, uint32_t parity, PfWaits* waits)
{
    unsigned long long t0 = 0, t;
    while (!__all_sync(0xffffffffu, mbar_poll(bar, parity)))
    {
        if (__any_sync(0xffffffffu, waits->aborted)) return false;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t0 == 0) t0 = t;
        else if (__any_sync(0xffffffffu, t - t0 > waits->limit_ns)) { waits->aborted = 1; return false; }
    }
    return true;
}
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, PfWaits* waits)
{
    if (__builtin_expect(__all_sync(0xffffffffu, mbar_poll(bar, parity)), 1)) return true;
    return wait_bar_slow(bar, parity, waits);
}
// (likewise mbar_wait_own)
__device__ __forceinline__ void wait_own(uint32_t bar, uint32_t parity)
{
    unsigned long long t0 = 0, t = 0;
    while (!__all_sync(0xffffffffu, mbar_poll(bar, parity)))
    {
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
        if (t0 == 0) t0 = t;
        else if (__any_sync(0xffffffffu, t - t0 > (unsigned long long)kPfWaitNs)) return;
    }
}
// a column of results, the first `there` of them
template <class O, int N>
__device__ __forceinline__ void store_column(O* to, long long stride, const uint64_t (&sum)[N], int there)
{
#pragma unroll
    for (int t = 0; t < 2 * N; ++t)
    {
        if (t < there) *to = from_float<O>(one_of(sum[t / 2], t & 1));
        to += stride;
    }
}
// all threads of the cluster, warp by warp
__device__ __forceinline__ void cluster_meet()
{
    tc_fence_before();
    __syncwarp();
    cluster_arrive();
    cluster_wait();
}

struct Wg {
    W4 w;
    int log_ck;
};

// a counter of stages with the parity of their barriers
template <int N>
struct Ring {
    uint32_t s = 0, parity = 0;
    __device__ __forceinline__ void next(uint32_t by = 1) { if ((s += by) >= N) { s -= N; parity ^= 1u; } }
};

template <class X, class SC, int GROUPS, int TOKENS>
__global__ void __launch_bounds__((WgPlan<GROUPS, TOKENS>::kThreads), 1) w4_gemm_kernel(const __grid_constant__ CUtensorMap map, Wg g)
{
    using Plan = WgPlan<GROUPS, TOKENS>;
    using Stream = typename Plan::Stream;
    constexpr int kStages = Plan::kStages;
    WgShared& sh = *reinterpret_cast<WgShared*>(wg_smem + Plan::kRest + Plan::kPlanes);
    const W4& a = g.w;
    uint8_t* const s_planes = wg_smem + Plan::kRest;
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int ck = 1 << g.log_ck, rank = blockIdx.x & (ck - 1);
    if (saddr(wg_smem) & 1023u)          // (never: the swizzled tiles would be read from the wrong places)
    {
        grid_dependency_wait();
        if (threadIdx.x == 0) atomicExch(a.status, 1);
        return;
    }
    const int c0 = (rank * a.C) >> g.log_ck, c1 = ((rank + 1) * a.C) >> g.log_ck, blocks = a.blocks;
    const bool zeros = a.zp != nullptr;
    if (threadIdx.x == 0)
    {
        for (int s = 0; s < kStages; ++s) { mbar_init(&sh.full_a[s], 8); mbar_init(&sh.full_b[s], 1); mbar_init(&sh.empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&sh.sum_full[s], 1); mbar_init(&sh.sum_empty[s], Plan::kSumWarps); }
        mbar_init(&sh.done, 1);
        sh.waits.aborted = 0; sh.waits.limit_ns = (unsigned long long)kPfWaitNs;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (a.start)
    {
        grid_dependency_wait();
        if (w4_other_call(a)) return;
    }
    if (warp == Plan::kMma)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    int passes;
    if (!a.start)
    {
        passes = (a.rows + TOKENS - 1) / TOKENS;
        if (threadIdx.x == 0) { sh.row[0] = sh.first[0] = 0; sh.row[1] = a.rows; sh.first[1] = passes; }
    }
    else
    {
        passes = expert_passes<TOKENS>(a, sh.row, sh.first, sh.warp_sums);
        zero_rows_behind(a, sh.row[a.E]);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(sh.tmem);
    const unsigned items = (unsigned)passes * blocks, clusters = gridDim.x >> g.log_ck, mine = blockIdx.x >> g.log_ck, each = items / clusters, more = items % clusters;
    const int i0 = mine * each + min(mine, more), i1 = i0 + each + (mine < more);
    W4Cursor now;
    now.seek(i0 < i1 ? i0 : 0, blocks, sh.first, a.E);
    // rows of x of an item
    auto rows_of = [&](const W4Cursor& c, int& base) {
        base = sh.row[c.e] + (c.pass - sh.first[c.e]) * TOKENS;
        return min(sh.row[c.e + 1] - base, TOKENS);
    };
    constexpr int kColumns = Plan::kColumns;
    if (warp < Plan::kSumWarps)
    {
        if (Plan::kSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
        // ---- sums
        const int quarter = warp & 3, t0 = (warp >> 2) * kColumns, r = quarter * 32 + lane;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + t0;
        uint64_t sum[kColumns / 2];                       // two tokens in each
        Ring<2> acc;
        uint32_t ready = 0;                               // the accumulator was there when last looked at
        bool ok = true;
        for (int i = i0; i < i1 && ok; ++i, now.next(blocks, sh.first, a.E, passes))
        {
            int base;
            const int rows = rows_of(now, base);
            const size_t unit = ((size_t)now.e * a.S + min(now.block * 8 + r / 16, a.S - 1)) * a.C;
            const uint16_t* sc = a.sc + (unit + c0) * 16 * GROUPS + (r & 7) * 2 * GROUPS + (r >> 3 & 1);
            // scales of the next chunks; a place is loaded again when its chunk is through (moved from place to place, a scale would be waited for by the move)
            constexpr int kAhead = GROUPS == 4 ? 2 : 4;
            uint16_t next[kAhead][GROUPS];
#pragma unroll
            for (int d = 0; d < kAhead; ++d)
#pragma unroll
                for (int j = 0; j < GROUPS; ++j) next[d][j] = c0 + d < c1 ? sc[d * 16 * GROUPS + 2 * j] : 0;
#pragma unroll
            for (int j = 0; j < kColumns / 2; ++j) sum[j] = 0;
#pragma unroll 1
            for (int c = c0; c < c1 && ok; c += kAhead)
#pragma unroll
                for (int d = 0; d < kAhead; ++d)
                {
                    if (c + d >= c1) break;
                    sc += 16 * GROUPS;
                    uint64_t scale[GROUPS];
#pragma unroll
                    for (int j = 0; j < GROUPS; ++j)
                    {
                        scale[j] = two_floats(scales_of<SC>(next[d][j]).x);
                        if (c + d + kAhead < c1) next[d][j] = sc[(kAhead - 1) * 16 * GROUPS + 2 * j];
                    }
#pragma unroll
                    for (int j0 = 0; j0 < GROUPS; j0 += Plan::kSet)
                    {
                        if (__builtin_expect(!__all_sync(0xffffffffu, ready), 0)) ok = ok && wait_bar_slow(saddr(&sh.sum_full[acc.s]), acc.parity, &sh.waits);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t at = from + acc.s * Plan::kSumColumns, sum_empty = saddr(&sh.sum_empty[acc.s]);
                        acc.next();
#pragma unroll
                        for (int j = 0; j < Plan::kSet; ++j)
                        {
                            uint32_t v[kColumns / 16][16];
#pragma unroll
                            for (int h = 0; h < kColumns / 16; ++h) tmem_ld16_async(at + j * TOKENS + 16 * h, v[h]);
#pragma unroll
                            for (int h = 0; h < kColumns / 16; ++h) tmem_wait_ld(v[h]);
                            if (j == Plan::kSet - 1)
                            {
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive32(sum_empty);
                                ready = mbar_test(saddr(&sh.sum_full[acc.s]), acc.parity);      // of the next accumulator, behind the products
                            }
#pragma unroll
                            for (int k = 0; k < kColumns / 2; ++k) fma_two(sum[k], scale[j0 + j], v[k / 8][2 * k % 16], v[k / 8][2 * k % 16 + 1]);
                        }
                    }
                    if (!ok) break;
                }
            if (ck == 1 && ok)
            {
                const int n = now.block * 128 + r, there = n < a.N ? rows - t0 : 0;
                const size_t first = (size_t)(base + t0) * a.out_stride + n;
                if (a.out_type == NQ_F32) store_column<float>((float*)a.out + first, a.out_stride, sum, there);
                else store_column<X>((X*)a.out + first, a.out_stride, sum, there);
            }
        }
        if (ck > 1)
        {
            // one item: when every CTA of the cluster is through with its tiles, their place takes the sums: [rank][token of the CTA's share][row]
            cluster_meet();
            const int log_share = 31 - __clz(TOKENS >> g.log_ck), share = 1 << log_share;
#pragma unroll
            for (int t = 0; t < kColumns; ++t)
            {
                const int token = t0 + t;
                const uint32_t at = cluster_address(saddr(wg_smem) + ((((rank << log_share) + (token & (share - 1))) << 7) + r) * 4, token >> log_share);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(one_of(sum[t / 2], t & 1)) : "memory");
            }
        }
    }
    else if (warp < Plan::kTma)
    {
        if (Plan::kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---- weights.  A warp reaches the quarter of tensor memory that its number has: strips 2 (warp % 4) and the one behind it.  Chunks are counted over all
        // items; of two warps to a strip one has the even ones, the other the odd ones.
        constexpr int kHalves = Plan::kHalves;
        const int who = warp - Plan::kSumWarps, strip = 2 * (warp & 3) + (who >> 2 & 1), half = who >> 3, chunks = c1 - c0;
        Stream planes((const char*)s_planes + who * Stream::kBytes, lane);
        W4Cursor ahead = now;
        int to_ask = i1 - i0, left = 0, parity = half;    // (parity: of the next item's first chunk that is this warp's)
        bool there = true;
        auto ask = [&] {
            while (--left < 0)
            {
                if (to_ask-- > 0)
                {
                    const int skip = kHalves == 2 ? parity : 0;
                    planes.seek(a, ((size_t)ahead.e * a.S + min(ahead.block * 8 + strip, a.S - 1)) * a.C + c0 + skip, lane);
                    ahead.next(blocks, sh.first, a.E, passes);
                    left = kHalves == 2 ? (chunks - skip + 1) >> 1 : chunks;
                    parity ^= chunks & 1;
                }
                else { there = false; left = 0x7fffffff; }
            }
            planes.ask(there, zeros);
        };
#pragma unroll 1
        for (int d = 0; d < Stream::kDepth; ++d) ask();
        const uint32_t to = tmem + ((uint32_t)(strip * 16) << 16) + 2 * Plan::kSumColumns;
        Ring<kStages> stage;
        stage.s = half;
        uint32_t stored = 0;                              // barrier of the unit whose stores are on their way
        for (int u = (i1 - i0) * chunks - half; u > 0; u -= kHalves)
        {
            W4Unit<GROUPS> unit;
            planes.oldest(unit, zeros);
            const uint32_t words[8] = {unit.w[0].x, unit.w[0].y, unit.w[0].z, unit.w[0].w, unit.w[1].x, unit.w[1].y, unit.w[1].z, unit.w[1].w};
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                uint32_t r[16];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    constexpr int kSteps = 8 / GROUPS;
                    const int group = (4 * h + j) / kSteps;
                    uint32_t lo, hi, f[4];
                    Operand<X>::zeros(unit.zp[group / 2] >> (16 * (group & 1)), lo, hi);
                    Operand<X>::weights(words[4 * h + j], lo, hi, f);
                    r[4 * j] = f[0]; r[4 * j + 1] = f[2]; r[4 * j + 2] = f[1]; r[4 * j + 3] = f[3];
                }
                if (h == 0)
                {
                    // the unit before this one has been stored by now
                    if (stored)
                    {
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive32(stored);
                    }
                    stored = 0;
                    if (!wait_bar(saddr(&sh.empty[stage.s]), stage.parity ^ 1u, &sh.waits)) { u = 0; break; }
                    tc_fence_after();
                }
                tmem_st_16x256b_x4(to + stage.s * 64 + h * 32, r);
            }
            if (u == 0) break;
            stored = saddr(&sh.full_a[stage.s]);
            ask();
            stage.next(kHalves);
        }
        if (stored)
        {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive32(stored);
        }
        copies_done<0>();
    }
    else
    {
    if (Plan::kSplit) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == Plan::kTma)
    {
        // ---- token tiles
        if (!a.start) grid_dependency_wait();
        const uint32_t tiles = saddr(wg_smem);
        Ring<kStages> stage;
        uint32_t asked = 0;                               // bit s: parity of the loads into stage s
        bool ok = true;
        for (int i = i0; i < i1 && ok; ++i, now.next(blocks, sh.first, a.E, passes))
        {
            int base;
            rows_of(now, base);
            for (int c = c0; c < c1; ++c)
            {
                ok = wait_bar(saddr(&sh.empty[stage.s]), stage.parity ^ 1u, &sh.waits);
                if (!ok) break;
                if (lane == 0) tma_two_boxes(tiles + stage.s * 2 * Plan::kBox, Plan::kBox, &map, c * 128, base, saddr(&sh.full_b[stage.s]));
                __syncwarp();
                asked ^= 1u << stage.s;
                stage.next();
            }
        }
        for (int s = 0; s < kStages; ++s) wait_own(saddr(&sh.full_b[s]), ((asked >> s) & 1u) ^ 1u);      // loads on their way
    }
    else if (warp == Plan::kMma)
    {
        // ---- MMAs
        constexpr uint32_t kType = std::is_same<X, __half>::value ? 0u : 1u;
        constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(TOKENS >> 3) << 17) | (8u << 24);      // fp32 sums, both operands K-major, M 128
        const uint64_t desc = smem_desc(saddr(wg_smem), 16, 1024, 2);
        const uint32_t b0 = (uint32_t)desc, b_hi = (uint32_t)(desc >> 32);
        // Stages and accumulators are constants here, so that the addresses are: what this warp issues beside the MMAs paces the kernel
        const uint32_t bars = saddr(&sh);
        uint32_t stage_parity = 0, sum_parity = 0;        // (of accumulator a: bit a)
        int left = (i1 - i0) * (c1 - c0);
        bool ok = true;
        auto chunk = [&](auto stage) {
            constexpr int kS = decltype(stage)::value, kSets = GROUPS / Plan::kSet, kFirstSum = kS * kSets & 1;
            constexpr int kA = offsetof(WgShared, full_a) + 8 * kS, kB = offsetof(WgShared, full_b) + 8 * kS, kEmpty = offsetof(WgShared, empty) + 8 * kS;
            if constexpr (kS < kStages)
            {
                if (left <= 0) return;
                // weights, tokens and an accumulator: three polls, one vote (a wait each, all of them complete, took 450 of 980 clocks a chunk)
                const uint32_t free_parity = ((sum_parity >> kFirstSum) & 1u) ^ 1u;
                uint32_t ready = mbar_poll(bars + kA, stage_parity);
                ready &= mbar_poll(bars + kB, stage_parity);
                ready &= mbar_poll(bars + offsetof(WgShared, sum_empty) + 8 * kFirstSum, free_parity);
                if (__builtin_expect(!__all_sync(0xffffffffu, ready), 0))
                    ok = wait_bar_slow(bars + kA, stage_parity, &sh.waits) && wait_bar_slow(bars + kB, stage_parity, &sh.waits) &&
                         wait_bar_slow(bars + offsetof(WgShared, sum_empty) + 8 * kFirstSum, free_parity, &sh.waits);
                const uint32_t w = tmem + 2 * Plan::kSumColumns + kS * 64, b_lo = b0 + kS * (2 * Plan::kBox >> 4);
                auto group = [&](auto j) {
                    constexpr int kJ = decltype(j)::value, kSteps = 8 / GROUPS, kFirst = kJ * kSteps;
                    if constexpr (kJ < GROUPS)
                    {
                        constexpr int kPlace = kJ % Plan::kSet, kSum = (kS * kSets + kJ / Plan::kSet) & 1;      // in the accumulator, and which
                        constexpr int kFree = offsetof(WgShared, sum_empty) + 8 * kSum, kFull = offsetof(WgShared, sum_full) + 8 * kSum;
                        if (kPlace == 0 && kJ) ok = ok && wait_bar(bars + kFree, ((sum_parity >> kSum) & 1u) ^ 1u, &sh.waits);
                        if (!ok) return;
                        if (kPlace == 0) tc_fence_after();
                        mma_group<kSteps, Plan::kBox, kPlace == Plan::kSet - 1, kJ == GROUPS - 1>(
                            tmem + kSum * Plan::kSumColumns + kPlace * TOKENS, w + kFirst * 8, b_lo + (kFirst >> 2) * (Plan::kBox >> 4) + (kFirst & 3) * 2, b_hi, kDesc,
                            bars + kFull, bars + kEmpty);
                        if (kPlace == Plan::kSet - 1) sum_parity ^= 1u << kSum;
                    }
                };
                group(std::integral_constant<int, 0>()); group(std::integral_constant<int, 1>()); group(std::integral_constant<int, 2>()); group(std::integral_constant<int, 3>());
                left = ok ? left - 1 : 0;
            }
        };
        static_assert(kStages % 2 == 0 && kStages <= 6, "a round of the stages leaves the accumulators where they were");
        while (left > 0)
        {
            chunk(std::integral_constant<int, 0>()); chunk(std::integral_constant<int, 1>()); chunk(std::integral_constant<int, 2>());
            chunk(std::integral_constant<int, 3>()); chunk(std::integral_constant<int, 4>()); chunk(std::integral_constant<int, 5>());
            stage_parity ^= 1u;
        }
        __syncwarp();
        tc_commit_elect(&sh.done);
        wait_own(saddr(&sh.done), 0);
    }
    }
    if (ck > 1 && warp >= Plan::kSumWarps) cluster_meet();
    launch_dependents();
    if (ck > 1)
    {
        const int share = TOKENS >> g.log_ck, log_share = 31 - __clz(share);
        cluster_meet();
        if (i0 < i1)
        {
            // (what every thread needs of the item)
            int base;
            W4Cursor item;
            item.seek(i0, blocks, sh.first, a.E);
            const int rows = rows_of(item, base);
            const float* part = reinterpret_cast<const float*>(wg_smem);
            for (int i = threadIdx.x; i < share * 128; i += blockDim.x)
            {
                const int token = (rank << log_share) + (i >> 7), n = item.block * 128 + (i & 127);
                if (token >= rows || n >= a.N) continue;
                float s = 0.f;
#pragma unroll 8
                for (int q = 0; q < ck; ++q) s += part[(q << (log_share + 7)) + i];
                store_as(a.out, a.out_type, (size_t)(base + token) * a.out_stride + n, s);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (sh.waits.aborted && threadIdx.x == 0) atomicExch(a.status, 1);
    if (warp == Plan::kMma) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// tensor map of rows of x [rows][K]: boxes of 64 columns x `tokens` rows, 128-byte swizzle, zeros behind the edges
int w4_x_map(CUtensorMap* map, const W4& a, int tokens, bool bf16)
{
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return fail(NQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[2] = {(cuuint64_t)a.K, (cuuint64_t)a.rows}, strides[1] = {(cuuint64_t)a.x_stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)tokens}, estr[2] = {1, 1};
    const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(a.x), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NQ_ERR_CUDA, "nq_w4_matmul: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return NQ_OK;
}

template <class X, class SC, int GROUPS, int TOKENS>
int wg_launch(Wg g, int device, cudaStream_t st)
{
    using Plan = WgPlan<GROUPS, TOKENS>;
    W4& a = g.w;
    CUtensorMap map;
    if (int e = w4_x_map(&map, a, TOKENS, std::is_same<X, __nv_bfloat16>::value)) return e;
    auto* kernel = w4_gemm_kernel<X, SC, GROUPS, TOKENS>;
    if (!allow_shared<w4_gemm_kernel<X, SC, GROUPS, TOKENS>>(Plan::kSmem, device)) return fail(NQ_ERR_CUDA, "nq_w4_matmul: shared memory");
    a.blocks = (a.S - 1) / 8 + 1;
    const int of = a.rows < a.upto ? a.rows : a.upto;          // rows that experts may have here
    const long long most = (long long)a.blocks * (a.start ? of / TOKENS + (a.E < of ? a.E : of) : (a.rows - 1) / TOKENS + 1);
    NQ_REQUIRE(most <= 0x7fffffff / a.C, "nq_w4_matmul: %d rows are too many", a.rows);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    cfg.blockDim = dim3(Plan::kThreads); cfg.dynamicSmemBytes = Plan::kSmem; cfg.stream = st;
    // columns are split while every item still has a cluster at once
    g.log_ck = 0;
    for (int log_ck = 1; !a.start && log_ck <= 3 && a.C >> log_ck >= 2 && most << log_ck <= a.sms; ++log_ck)
    {
        attr[0].val.clusterDim.x = 1 << log_ck;
        if (most > active_clusters<w4_gemm_kernel<X, SC, GROUPS, TOKENS>>(1 << log_ck, device, cfg)) break;
        g.log_ck = log_ck;
    }
    attr[0].val.clusterDim.x = 1 << g.log_ck;
    cfg.numAttrs = 2;
    const long long clusters = g.log_ck ? most : most < a.sms ? most : a.sms;
    cfg.gridDim = dim3((unsigned)(clusters << g.log_ck));
    cudaLaunchKernelEx(&cfg, kernel, map, g);
    return check_launch("nq_w4_matmul");
}
template <class X, class SC, int GROUPS>
int wg_tokens(const Wg& g, int tokens, int device, cudaStream_t st)
{
    return tokens == 32 ? wg_launch<X, SC, GROUPS, 32>(g, device, st) : tokens == 64 ? wg_launch<X, SC, GROUPS, 64>(g, device, st) : wg_launch<X, SC, GROUPS, 128>(g, device, st);
}
template <class X, class SC>
int wg_groups(const Wg& g, int tokens, int group, int device, cudaStream_t st)
{
    return group == 128 ? wg_tokens<X, SC, 1>(g, tokens, device, st) : group == 64 ? wg_tokens<X, SC, 2>(g, tokens, device, st) : wg_tokens<X, SC, 4>(g, tokens, device, st);
}

// with items of `tokens` rows of x: 32, 64 or 128
int w4_gemm(const W4& a, int tokens, int type, int sc_type, int group, int device, cudaStream_t st)
{
    const Wg g{a, 0};
    if (type == NQ_F16) return sc_type == NQ_F16 ? wg_groups<__half, __half>(g, tokens, group, device, st) : wg_groups<__half, __nv_bfloat16>(g, tokens, group, device, st);
    return sc_type == NQ_F16 ? wg_groups<__nv_bfloat16, __half>(g, tokens, group, device, st) : wg_groups<__nv_bfloat16, __nv_bfloat16>(g, tokens, group, device, st);
}

}  // namespace nq
