// Products with 4-bit weights (nq_w4.cuh): the layout of the planes, and the kernel for calls of few rows.
#include <limits.h>

#include "nq_tc.cuh"
#include "nq_w4.cuh"

namespace nq {

// ---- layout -------------------------------------------------------------------------------------------------------------------

struct W4Layout {
    const uint8_t* q; const uint16_t* scales; const uint8_t* zeros;      // [E][N][K / 2], [E][N][K / g] x 2
    uint32_t* qw; uint16_t* sc; uint8_t* zp;
    int E, N, K, g, S, C;
};

// a thread per word of the units, kLayoutUnits of them; the first threads of a unit write its scales too.  Neighbouring threads read 32 bytes of a row together: 403 MB
// of weights in 0.37 ms (byte by byte: 0.95).
constexpr int kLayoutUnits = 4;
__global__ void __launch_bounds__(256) w4_layout_kernel(W4Layout a, unsigned units)
{
    const int word4 = threadIdx.x, lane = word4 / 4 % 32, word = (word4 / 128) * 4 + word4 % 4, g = lane / 4, t = lane % 4;
    const unsigned first = blockIdx.x * kLayoutUnits;
    uint32_t pair[kLayoutUnits][2];                       // the lane's four columns of rows g and g + 8, as they are: 8 is a weight of 0
#pragma unroll
    for (int i = 0; i < kLayoutUnits; ++i)
    {
        const unsigned unit = first + i, strip = unit / a.C, c = unit - strip * a.C, e = strip / a.S;      // (e S + strip) C + chunk
        const int k = (int)c * 128 + word * 16 + 4 * t, row = (int)(strip - e * a.S) * 16 + g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            pair[i][h] = 0x8888u;
            if (unit < units && row + 8 * h < a.N && k < a.K) pair[i][h] = *reinterpret_cast<const uint16_t*>(a.q + ((size_t)e * a.N + row + 8 * h) * (a.K / 2) + k / 2);
        }
    }
#pragma unroll
    for (int i = 0; i < kLayoutUnits; ++i)
    {
        const unsigned unit = first + i;
        if (unit >= units) return;
        // columns 0, 1, 2, 3 of a row to nibbles 0, 4, 2, 6; of the other row to those behind them
        auto spread = [](uint32_t v) { return (v & 15u) | (v & 0xf0u) << 12 | (v & 0xf00u) | (v & 0xf000u) << 12; };
        a.qw[(size_t)unit * 256 + word4] = spread(pair[i][0]) | spread(pair[i][1]) << 4;
        const int per = 128 / a.g, groups = a.K / a.g;    // groups of a unit, of a row
        if (word4 < 16 * per)
        {
            const unsigned strip = unit / a.C, c = unit - strip * a.C, e = strip / a.S;
            const int r = (int)(strip - e * a.S) * 16 + word4 / (2 * per) + 8 * (word4 & 1), j = (int)c * per + word4 / 2 % per;
            const bool in = r < a.N && j < groups;
            const size_t from = ((size_t)e * a.N + r) * groups + j, to = (size_t)unit * 16 * per + word4;
            a.sc[to] = in ? a.scales[from] : 0;
            if (a.zp) a.zp[to] = in ? a.zeros[from] & 15 : 8;
        }
    }
}

// Products of a single matrix ask for planes before their predecessor's end has been waited for, when its writes need not be there.  Nothing starts this kernel early,
// so that the layout's are when it runs.
__global__ void w4_settled_kernel() {}

// ---- product ------------------------------------------------------------------------------------------------------------------

// acc += the unit's 16 x 128 weights times rows of x: xs[n] = shared address of the lane's row of tile n, its pieces of the unit's columns
template <class X, class SC, int GROUPS, int TILES>
__device__ __forceinline__ void unit_product(const W4Unit<GROUPS>& u, const uint32_t (&xs)[TILES], float (&acc)[TILES][4])
{
    const uint32_t words[8] = {u.w[0].x, u.w[0].y, u.w[0].z, u.w[0].w, u.w[1].x, u.w[1].y, u.w[1].z, u.w[1].w};
#pragma unroll
    for (int j = 0; j < GROUPS; ++j)
    {
        uint32_t lo, hi;
        Operand<X>::zeros(u.zp[j / 2] >> (16 * (j & 1)), lo, hi);
        float part[TILES][4];
#pragma unroll
        for (int q = 0; q < 4 / GROUPS; ++q)
        {
            const int G = j * (4 / GROUPS) + q;
            uint32_t a0[4], a1[4];
            Operand<X>::weights(words[2 * G], lo, hi, a0);
            Operand<X>::weights(words[2 * G + 1], lo, hi, a1);
#pragma unroll
            for (int n = 0; n < TILES; ++n)
            {
                const uint4 b = load_shared16(xs[n] + G * 64);
                if (q == 0) Operand<X>::template mma<true>(part[n], a0, b.x, b.y);
                else Operand<X>::template mma<false>(part[n], a0, b.x, b.y);
                Operand<X>::template mma<false>(part[n], a1, b.z, b.w);
            }
        }
        const float2 sc = scales_of<SC>(u.sc[j]);
#pragma unroll
        for (int n = 0; n < TILES; ++n)
        {
            acc[n][0] += sc.x * part[n][0]; acc[n][1] += sc.x * part[n][1];
            acc[n][2] += sc.y * part[n][2]; acc[n][3] += sc.y * part[n][3];
        }
    }
}

// shared memory of a CTA
template <int GROUPS, int TILES>
struct W4Plan {
    using Stream = W4Stream<GROUPS, 4>;
    static constexpr int kPitch = 8 * TILES + 2, kPart = kW4Warps * 16 * kPitch;
    // parts of two items: the sums of one wait for the next one's products
    static constexpr int kPlanes = kW4Warps * Stream::kBytes, kParts = 2 * kPart * 4, kRoom = kW4MaxShared - kPlanes - kParts;      // for rows of x
};

// A warp's share of an item: its part of the columns of one strip times the item's rows, while it asks for what comes kDepth units later
template <class X, class SC, int GROUPS, int TILES, int MOST, class STREAM, class NEXT>
__device__ __forceinline__ void strip_product(STREAM& planes, int units, bool zeros, uint32_t x0, int pitch, int rows, int lane,
                                              float (&acc)[MOST][4], NEXT&& ask)
{
    // columns of a tile behind the last row read that row again: nobody looks at what comes of them
    uint32_t xs[TILES];
#pragma unroll
    for (int n = 0; n < TILES; ++n) xs[n] = x0 + min(8 * n + (lane >> 2), rows - 1) * pitch + (lane & 3) * 16;
    float sum[TILES][4] = {};
#pragma unroll 4
    for (int u = 0; u < units; ++u)
    {
        W4Unit<GROUPS> unit;
        planes.oldest(unit, zeros);
        unit_product<X, SC, GROUPS, TILES>(unit, xs, sum);
#pragma unroll
        for (int n = 0; n < TILES; ++n) xs[n] += 256;
        ask();
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = sum[n][i];
}

// For calls of up to 16 rows: bound by HBM by intent, by the instructions that unpack the weights in practice.  A unit costs a warp 152 instructions (32 masks, 8 shifts,
// 32 half-pair additions, 8 MMAs; 57 of them on the half-rate integer pipe, 20 for a share of its item's sums), four warps of a scheduler issue in two thirds of the
// clocks.  us, captured, one launch after the other, 1 / 8 / 16 rows of 4,096 x 6,144 (floor 2.0): 5.7 / 7.6 / 9.5; one row of 32,768 x 8,192 31 (4.5 TB/s;
// floor 21), of 16 x 128 2.4.  What made the difference, one row of 32,768 x 8,192: units asked for ahead into registers 57 (their loads shared the few scoreboards);
// through shared memory, a CTA per block of strips 55; one CTA per SM with units asked for across items 43; cuts in shifts instead of 64-bit divisions 39; masks as one
// instruction each 34; cuts by rounds 32; predicates instead of branches 31.  32 warps of 64 registers: 35.
//
// One CTA per SM, in clusters of `ck` that split the matrix into ranges of columns, each taking a run of consecutive items.  A block has ws = 16 / wk strips, wk
// warps for each: part p = rank wk + warp % wk of parts = ck wk multiplies the units [p C / parts, (p + 1) C / parts) of its strip with up to 8 TILES rows
// of x, which stay in shared memory as long as the rows are the same.  Units are asked for across the borders of items, so that memory does not
// wait for sums.  Each CTA of a cluster adds up ws 16 / ck rows of the result: the warps store their parts of those into its shared memory, one
// barrier per item, whose sums are taken after the next item's products.  The parts are added in their order: the same call gives the same bits.
template <class X, class SC, int GROUPS, int TILES>
__global__ void __launch_bounds__(32 * kW4Warps, 1) w4_kernel(W4 a)
{
    using Plan = W4Plan<GROUPS, TILES>;
    using Stream = typename Plan::Stream;
    constexpr int kRows = 8 * TILES, kPitch = Plan::kPitch;
    // [warp] Stream; [2][part][row of the matrix][row of x] of this CTA's rows, for two items; rows of x, a.pitch apart
    extern __shared__ __align__(16) char s_planes[];
    __shared__ int s_row[kW4MaxExperts + 1], s_first[kW4MaxExperts + 2], s_warp[32];       // experts' rows of x, first passes
    float* const s_part = reinterpret_cast<float*>(s_planes + Plan::kPlanes);
    char* const s_x = s_planes + Plan::kPlanes + Plan::kParts;
    const int lane = threadIdx.x & 31, warp = (int)uniform(threadIdx.x >> 5), g = lane >> 2, t = lane & 3;
    const int ck = 1 << a.log_ck, wk = 1 << a.log_wk, ws = kW4Warps >> a.log_wk, log_parts = a.log_ck + a.log_wk, blocks = a.blocks;
    const int rank = blockIdx.x & (ck - 1), w = warp & (wk - 1), in_block = warp >> a.log_wk, p = (rank << a.log_wk) + w;
    const int u0 = (p * a.C) >> log_parts, units = (((p + 1) * a.C) >> log_parts) - u0;
    const int c0 = (rank * a.C) >> a.log_ck, c1 = ((rank + 1) * a.C) >> a.log_ck;      // units of the CTA's rows of x
    const bool zeros = a.zp != nullptr;
    int passes;
    if (!a.start)
    {
        passes = (a.rows + kRows - 1) / kRows;
        if (threadIdx.x == 0) { s_row[0] = s_first[0] = 0; s_row[1] = a.rows; s_first[1] = passes; }
        __syncthreads();
    }
    else
    {
        grid_dependency_wait();
        if (w4_other_call(a)) return;
        passes = expert_passes<kRows>(a, s_row, s_first, s_warp);
        zero_rows_behind(a, s_row[a.E]);
    }
    // as many items for each cluster, one more for the first ones
    const unsigned items = (unsigned)passes * blocks, clusters = gridDim.x >> a.log_ck, mine = blockIdx.x >> a.log_ck, each = items / clusters, more = items % clusters;
    const int i0 = mine * each + min(mine, more), i1 = i0 + each + (mine < more);
    if (i0 == i1)                                         // the whole cluster
    {
        if (!a.start) grid_dependency_wait();
        launch_dependents();
        return;
    }
    Stream planes(s_planes + warp * Stream::kBytes, lane);
    W4Cursor now, ahead;
    now.seek(i0, blocks, s_first, a.E);
    ahead = now;
    int to_ask = i1 - i0, in_strip = 0;      // items to ask for, units left of the present one
    bool there = true;
    auto ask = [&] {
        if (--in_strip < 0)
        {
            if (to_ask-- > 0)
            {
                // (strips behind the last one: that one again, nobody looks at what comes of it)
                planes.seek(a, ((size_t)ahead.e * a.S + min(ahead.block * ws + in_block, a.S - 1)) * a.C + u0, lane);
                ahead.next(blocks, s_first, a.E, passes);
                in_strip = units - 1;
            }
            else { there = false; in_strip = 0x7fffffff; }
        }
        planes.ask(there, zeros);
    };
    // the planes do not come from a kernel that lets its successors in early: those of a single matrix are asked for before the wait.  Half of the ring
    // first, then the rows of x, then the other half, which need not be there when the products begin.
    constexpr int kDepth = Stream::kDepth, kBefore = kDepth / 2;
#pragma unroll 1
    for (int d = 0; d < kBefore; ++d) ask();
    if (!a.start) grid_dependency_wait();
    launch_dependents();
    if (ck > 1) cluster_arrive();                       // the others' shared memory is there when all have come by
    const int log_own = 8 - a.log_wk - a.log_ck, own = 1 << log_own;       // rows of the matrix whose sums this CTA adds up: ws 16 / ck
    // the sums of an item whose parts have been stored, after the barrier
    auto add_up = [&](const float* part, int block, int base, int rows) {
        for (int i = threadIdx.x; i < rows * own; i += blockDim.x)
        {
            const int r = i >> log_own, n = i & (own - 1), to = block * ws * 16 + rank * own + n;
            float sum = 0.f;
#pragma unroll 8
            for (int q = 0; q < 1 << log_parts; ++q) sum += part[((q << log_own) + n) * kPitch + r];
            if (to < a.N) store_as(a.out, a.out_type, (size_t)(base + r) * a.out_stride + to, sum);
        }
    };
    auto barrier = [&] {
        if (ck > 1) cluster_wait();
        else __syncthreads();
    };
    int old_block = -1, old_base = 0, old_rows = 0, pass = -1, base = 0, rows = 0;
    for (int i = i0; i < i1; ++i)
    {
        if (now.pass != pass)
        {
            // other rows of x: pieces of 128 columns, in turn to the warps
            pass = now.pass;
            base = s_row[now.e] + (pass - s_first[now.e]) * kRows;
            rows = min(s_row[now.e + 1] - base, kRows);
            __syncthreads();
            const int pieces = c1 - c0;
            for (int r = 0, c = warp; r < rows; c += kW4Warps)
            {
                while (c >= pieces) { c -= pieces; ++r; }
                // four columns a lane; a lane's four columns of two steps side by side
                const int k = (c0 + c) * 128 + lane * 4, there = k < a.K ? 8 : 0;            // zeros behind the last column
                const uint32_t to = shared_address(s_x) + r * a.pitch + c * 256 + (lane >> 3) * 64 + (lane & 3) * 16 + (lane >> 2 & 1) * 8;
                if (r < rows)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" :: "r"(to), "l"((const X*)a.x + (size_t)(base + r) * a.x_stride + (there ? k : 0)), "r"(there) : "memory");
            }
            copies_end();
            if (i == i0)
            {
#pragma unroll 1
                for (int d = kBefore; d < kDepth; ++d) ask();
                copies_done<kDepth - kBefore>();
            }
            else copies_done<0>();                        // (and the units that were asked for before)
            __syncthreads();
        }
        const uint32_t x0 = shared_address(s_x) + (u0 - c0) * 256;
        float acc[TILES][4];
        if (TILES == 2 && rows <= 8) strip_product<X, SC, GROUPS, 1>(planes, units, zeros, x0, a.pitch, rows, lane, acc, ask);
        else strip_product<X, SC, GROUPS, TILES>(planes, units, zeros, x0, a.pitch, rows, lane, acc, ask);
        // all parts of the item before this one are there, and those of the one before that have been read
        if (i > i0 || ck > 1) barrier();
        if (i > i0) add_up(s_part + ((i - 1) & 1) * Plan::kPart, old_block, old_base, old_rows);
        const uint32_t to = shared_address(s_part + (i & 1) * Plan::kPart);
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const int n = in_block * 16 + 8 * h + g, owner = n >> log_own;
            const uint32_t at = cluster_address(to + (((p << log_own) + (n & (own - 1))) * kPitch + 2 * t) * 4, owner);
#pragma unroll
            for (int q = 0; q < TILES; ++q)
                if (q == 0 || 8 * q < rows) cluster_store(at + 32 * q, acc[q][2 * h], acc[q][2 * h + 1]);
        }
        if (ck > 1) cluster_arrive();
        old_block = now.block; old_base = base; old_rows = rows;
        now.next(blocks, s_first, a.E, passes);
    }
    barrier();
    add_up(s_part + ((i1 - 1) & 1) * Plan::kPart, old_block, old_base, old_rows);
}

int w4_gemm(const W4& a, int tokens, int type, int sc_type, int group, int device, cudaStream_t st);       // nq_w4_gemm.cu

bool w4_shape(int E, int N, int K, int g)
{
    return E >= 1 && E <= kW4MaxExperts && N >= 1 && K <= kW4MaxColumns && (g == 32 || g == 64 || g == 128) && K >= g && K % g == 0;
}
// a copy takes the zero points of two rows in a unit: 8 bytes with groups of 32, 4 with others (of 128: two more rows' with them)
bool w4_zeros_aligned(const void* zp, int g) { return reinterpret_cast<uintptr_t>(zp) % (g == 32 ? 8 : 4) == 0; }
int w4_strips(int N) { return (N - 1) / 16 + 1; }
int w4_chunks(int K) { return (K - 1) / 128 + 1; }

// bytes between rows of x in shared memory: 64 off a multiple of 128, so that two rows of a fragment share the banks
int w4_pitch(int C, int ck) { return ((C + ck - 1) / ck) * 256 + 64; }

// How a matrix is cut: CTAs of a cluster and warps of a CTA that share a strip, both powers of two.  The device takes ceil(blocks / clusters) rounds; a round
// costs a warp its units and what comes per item (sums and barriers: as much as a unit and a half, over a cluster three).  Rows of x weigh in so that 8 rows of
// 6,144 columns, 98 KB for each CTA of its own, are shared by two CTAs: 7.6 us instead of 8.2.
template <class X, class SC, int GROUPS, int TILES>
bool w4_cut(W4& a, int rows, int device, cudaLaunchConfig_t& cfg, long long& clusters)
{
    using Plan = W4Plan<GROUPS, TILES>;
    const int experts = a.E < 8 ? a.E : 8;                // (taken to have rows)
    double best = 0;
    for (int log_ck = 0; log_ck <= 3; ++log_ck)
    {
        const int ck = 1 << log_ck;
        if (ck > a.C || rows * w4_pitch(a.C, ck) > Plan::kRoom) continue;
        cudaLaunchAttribute& cluster = cfg.attrs[0];
        cluster.val.clusterDim.x = ck;
        cfg.dynamicSmemBytes = Plan::kPlanes + Plan::kParts + (size_t)rows * w4_pitch(a.C, ck);
        const int there = ck == 1 ? a.sms : active_clusters<w4_kernel<X, SC, GROUPS, TILES>>(ck, device, cfg);
        for (int log_wk = 0; log_wk <= 4 && ck << log_wk <= a.C; ++log_wk)
        {
            const int blocks = (a.S - 1) / (kW4Warps >> log_wk) + 1, units = ((a.C - 1) >> (log_ck + log_wk)) + 1;
            // (16 units, one for each warp, come through the same door as 16 KB of x)
            const double cost = (((long long)blocks * experts - 1) / there + 1) * (units + (ck > 1 ? 3.0 : 1.5)) + rows * w4_pitch(a.C, ck) / 16384.0;
            if (best == 0 || cost < best)
            {
                best = cost;
                a.log_ck = log_ck; a.log_wk = log_wk; a.blocks = blocks; a.pitch = w4_pitch(a.C, ck);
                clusters = there;
            }
        }
    }
    return best > 0;
}

template <class X, class SC, int GROUPS, int TILES>
int w4_launch(W4 a, int device, cudaStream_t st)
{
    using Plan = W4Plan<GROUPS, TILES>;
    const int rows = a.rows < 8 * TILES ? a.rows : 8 * TILES;
    auto* kernel = w4_kernel<X, SC, GROUPS, TILES>;
    if (!allow_shared<w4_kernel<X, SC, GROUPS, TILES>>(kW4MaxShared, device)) return fail(NQ_ERR_CUDA, "nq_w4_matmul: shared memory");
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    cfg.blockDim = dim3(32 * kW4Warps); cfg.stream = st;
    long long clusters;
    if (!w4_cut<X, SC, GROUPS, TILES>(a, rows, device, cfg, clusters)) return fail(NQ_ERR_ARG, "nq_w4_matmul: no room for %d rows of %d columns", rows, a.K);
    const int of = a.rows < a.upto ? a.rows : a.upto;          // rows that experts may have here
    const long long most = (long long)a.blocks * (a.start ? of / (8 * TILES) + (a.E < of ? a.E : of) : (a.rows - 1) / (8 * TILES) + 1);
    NQ_REQUIRE(most <= 0x7fffffff / a.C, "nq_w4_matmul: %d rows are too many", a.rows);       // (units are counted in 32 bits)
    if (most < clusters) clusters = most;
    attr[0].val.clusterDim.x = 1 << a.log_ck;
    cfg.gridDim = dim3((unsigned)(clusters << a.log_ck));
    cfg.dynamicSmemBytes = Plan::kPlanes + Plan::kParts + (size_t)rows * a.pitch;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kernel, a);
    return check_launch("nq_w4_matmul");
}
template <class X, class SC, int GROUPS>
int w4_tiles(const W4& a, int device, cudaStream_t st)
{
    // one tile of eight rows where the call has no more, or an expert on average, or shared memory does not hold sixteen; else two
    if (a.start || a.rows <= 8 || 16 * w4_pitch(a.C, a.C < 8 ? a.C : 8) > W4Plan<GROUPS, 2>::kRoom) return w4_launch<X, SC, GROUPS, 1>(a, device, st);
    return w4_launch<X, SC, GROUPS, 2>(a, device, st);
}
template <class X, class SC>
int w4_groups(const W4& a, int g, int device, cudaStream_t st)
{
    return g == 128 ? w4_tiles<X, SC, 1>(a, device, st) : g == 64 ? w4_tiles<X, SC, 2>(a, device, st) : w4_tiles<X, SC, 4>(a, device, st);
}
int w4_few(const W4& a, int type, int sc_type, int group, int device, cudaStream_t st)
{
    if (type == NQ_F16) return sc_type == NQ_F16 ? w4_groups<__half, __half>(a, group, device, st) : w4_groups<__half, __nv_bfloat16>(a, group, device, st);
    return sc_type == NQ_F16 ? w4_groups<__nv_bfloat16, __half>(a, group, device, st) : w4_groups<__nv_bfloat16, __nv_bfloat16>(a, group, device, st);
}

}  // namespace nq

extern "C" {

int nq_w4_units(int E, int N, int K, int64_t* units)
{
    NQ_REQUIRE(units && nq::w4_shape(E, N, K, 32), "nq_w4_units: E = %d, N = %d, K = %d", E, N, K);
    *units = (int64_t)E * nq::w4_strips(N) * nq::w4_chunks(K);
    return NQ_OK;
}

int nq_w4_layout(const void* q, const void* scales, const void* zeros, int E, int N, int K, int group, void* qw, void* sc, void* zp, void* stream)
{
    NQ_REQUIRE(nq::w4_shape(E, N, K, group), "nq_w4_layout: E = %d, N = %d, K = %d, group = %d (32, 64 or 128, a divisor of K)", E, N, K, group);
    NQ_REQUIRE(q && scales && qw && sc && !zeros == !zp && nq::aligned16(qw) && nq::aligned16(sc) && nq::aligned_to(2, {q, scales}),
               "nq_w4_layout: null or unaligned pointer");
    NQ_REQUIRE(nq::w4_zeros_aligned(zp, group), "nq_w4_layout: zero points start on 8 bytes (groups of 32) or 4");
    const int S = nq::w4_strips(N), C = nq::w4_chunks(K);
    NQ_REQUIRE((int64_t)E * S * C <= 0x7fffffff, "nq_w4_layout: too many units");
    const unsigned units = (unsigned)((int64_t)E * S * C);
    nq::w4_layout_kernel<<<(units - 1) / nq::kLayoutUnits + 1, 256, 0, (cudaStream_t)stream>>>(nq::W4Layout{(const uint8_t*)q, (const uint16_t*)scales, (const uint8_t*)zeros, (uint32_t*)qw, (uint16_t*)sc, (uint8_t*)zp, E, N, K, group, S, C}, units);
    nq::w4_settled_kernel<<<1, 1, 0, (cudaStream_t)stream>>>();
    return nq::check_launch("nq_w4_layout");
}

int nq_w4_matmul(const void* x, int type, long long x_stride, const void* qw, const void* sc, int sc_type, const void* zp, const int32_t* start, int rows, int E,
                 int N, int K, int group, void* out, int out_type, long long out_stride, int32_t* status, void* stream)
{
    NQ_REQUIRE(nq::w4_shape(E, N, K, group) && rows >= 0, "nq_w4_matmul: rows = %d, E = %d, N = %d, K = %d, group = %d", rows, E, N, K, group);
    NQ_REQUIRE((type == NQ_F16 || type == NQ_BF16) && (sc_type == NQ_F16 || sc_type == NQ_BF16) && (out_type == type || out_type == NQ_F32),
               "nq_w4_matmul: types %d, %d -> %d", type, sc_type, out_type);
    NQ_REQUIRE(start || E == 1, "nq_w4_matmul: %d matrices without the rows' start array", E);
    NQ_REQUIRE(x_stride >= K && out_stride >= N, "nq_w4_matmul: row strides %lld, %lld", x_stride, out_stride);
    if (rows == 0) return NQ_OK;
    NQ_REQUIRE(x && qw && sc && out && status, "nq_w4_matmul: null pointer");
    NQ_REQUIRE(nq::aligned16(x) && x_stride % 8 == 0 && nq::aligned16(qw) && nq::aligned16(sc), "nq_w4_matmul: rows of x and planes start on 16 bytes");
    NQ_REQUIRE(nq::aligned_to(4, {start, status}) && nq::aligned_to(nq::type_size(out_type), {out}), "nq_w4_matmul: pointers are not aligned to the elements");
    NQ_REQUIRE(nq::w4_zeros_aligned(zp, group), "nq_w4_matmul: zero points start on 8 bytes (groups of 32) or 4");
    nq::W4 a{(const uint4*)qw, (const uint16_t*)sc, (const uint8_t*)zp, x, start, out, status, x_stride, out_stride, rows, N, K, E, nq::w4_strips(N), nq::w4_chunks(K),
             out_type, 0, 0, 0, 0, 0, -1, INT_MAX};
    int device;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&a.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
        return nq::fail(NQ_ERR_CUDA, "nq_w4_matmul: no device");
    cudaStream_t st = (cudaStream_t)stream;
    // This kernel or that of nq_w4_gemm.cu, us: 9.0 / 9.5 with 12 rows of 4,096 x 6,144, 9.4 / 9.5 with 16, 15.4 / 9.7 with 32 (four tiles here); of 6,144 x 2,048 in groups of
    // 64, 7.5 / 7.2, 7.7 / 7.3, 11.4 / 7.4; of 16,384 x 8,192, 24.9 / 25.1, 26.7 / 25.1.
    if (!start) return rows > 16 ? nq::w4_gemm(a, rows <= 32 ? 32 : rows <= 64 ? 64 : 128, type, sc_type, group, device, st) : nq::w4_few(a, type, sc_type, group, device, st);
    // Experts' numbers of rows differ, and one of nine takes two passes here.  32 experts of 4,096 x 6,144 with 4, 8, 12 rows on average: 95 / 111, 136 / 132, 155 / 133;
    // 128 of 2,048 x 2,048: 68 / 71, 101 / 81, 129 / 94; 64 of 2,048 x 4,096 in groups of 32: 75 / 92, 108 / 101, 117 / 107.  There, an expert of one and a half times the
    // average should not take two passes, of 32, 64 or 128 rows.  A launch that ends at once costs 0.5 us here, 2.3 there: the one for items of 32 rows is made
    // in the place of others for 64 MB of planes or more, which take 20 or longer (an eighth of 64 and 128 rows for each of the 32 experts: 170 -> 133, 200 -> 155).
    const int few = 8 * E, some = 64 * E / 3, tokens = rows <= some ? 32 : rows <= 2 * some ? 64 : 128;
    auto launch = [&](int form, int upto) {
        a.upto = rows <= upto ? INT_MAX : upto;
        const int e = form ? nq::w4_gemm(a, form, type, sc_type, group, device, st) : nq::w4_few(a, type, sc_type, group, device, st);
        a.more = a.upto;
        return e;
    };
    int e = launch(0, few);
    if (!e && a.more != INT_MAX && tokens > 32 && (int64_t)E * a.S * a.C >= 65536) e = launch(32, some);
    if (!e && a.more != INT_MAX) e = launch(tokens, INT_MAX);
    return e;
}

}  // extern "C"
