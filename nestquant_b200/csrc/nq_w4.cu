// Products with 4-bit weights that have a scale and a zero point per row and group of 32, 64 or 128 columns:
//   y[r][n] = sum over groups j of s[n][j] sum_{k in j} (q[n][k] - z[n][j]) x[r][k]
// for one matrix, or for one matrix per expert and rows that are sorted by expert.
//
// Layout (nq_w4_layout, once per matrix): units of 16 rows x 128 columns, 1 KB each, unit index (strip C + chunk), as the packed planes of
// the experts.  A unit is eight steps of m16n8k16, weights as A; inside a group of 32 columns lane (g, t) = (lane / 4, lane % 4) has the columns
// 8 t .. 8 t + 7, four for each of two steps, so that its tokens' operand is 16 consecutive bytes of a plain row of x, and no step crosses a
// group.  A lane's 32-bit word of a step holds, by nibble: 0, 4 = row g, columns 0, 1 of the step's four; 1, 5 = row g + 8, columns 0, 1; 2, 6 and
// 3, 7 the same rows, columns 2, 3: each pair is one masked word away from a pair of halves.  Word w of lane i sits at
// ((w / 4) 32 + i) 16 + (w % 4) 4 of the unit.  Scales [unit][g][group of the unit][row g, row g + 8], zero points likewise as bytes.
// Rows and columns behind the matrix have scale 0.
//
// q - z is exact in fp16 and in bf16 (integers to 15 in magnitude), products and sums of a group are in 32 bits on the tensor pipe, and
// the group's scale is applied to its sum in 32 bits: nothing is rounded to fewer bits before the result.
#include <atomic>
#include <type_traits>

#include "nq_common.cuh"
#include "nq_scan.cuh"
#include "nq_types.cuh"

namespace nq {

constexpr int kW4Warps = 16, kW4MaxExperts = 1024;
constexpr int kW4MaxShared = 216 * 1024;      // planes, rows of x and partial sums, beside the experts' rows
constexpr int kW4MaxColumns = 32768;          // eight rows of x in a cluster of eight: 66 KB

struct W4 {
    const uint4* qw; const uint16_t* sc; const uint8_t* zp;
    const void* x; const int* start; void* out;
    long long x_stride, out_stride;
    int rows, N, K, E, S, C, out_type;
    int log_ck, log_wk, pitch, blocks, sms;         // see w4_kernel
};

// ---- layout -------------------------------------------------------------------------------------------------------------------

struct W4Layout {
    const uint8_t* q; const uint16_t* scales; const uint8_t* zeros;      // [E][N][K / 2], [E][N][K / g] x 2
    uint32_t* qw; uint16_t* sc; uint8_t* zp;
    int E, N, K, g, S, C;
};

// a thread per word of the units; the first threads of a unit write its scales too
__global__ void __launch_bounds__(256) w4_layout_kernel(W4Layout a)
{
    const size_t unit = blockIdx.x;                       // (e S + strip) C + chunk
    const int w4 = threadIdx.x, c = (int)(unit % a.C), s = (int)(unit / a.C % a.S), e = (int)(unit / a.C / a.S);
    const int lane = w4 / 4 % 32, word = (w4 / 128) * 4 + w4 % 4, g = lane / 4, t = lane % 4;
    const int k0 = c * 128 + (word / 2) * 32 + 8 * t + 4 * (word % 2);
    const uint8_t* q = a.q + (size_t)e * a.N * (a.K / 2);
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        const int row = s * 16 + g + 8 * (i & 1), k = k0 + 2 * ((i >> 1) & 1) + (i >> 2);
        uint32_t n = 8;
        if (row < a.N && k < a.K) n = q[(size_t)row * (a.K / 2) + k / 2] >> (4 * (k & 1)) & 15;
        v |= n << (4 * i);
    }
    a.qw[unit * 256 + w4] = v;
    const int per = 128 / a.g, groups = a.K / a.g;        // groups of a unit, of a row
    if (w4 < 16 * per)
    {
        const int r = s * 16 + w4 / (2 * per) + 8 * (w4 & 1), j = c * per + w4 / 2 % per;
        const bool in = r < a.N && j < groups;
        const size_t from = ((size_t)e * a.N + r) * groups + j, to = unit * 16 * per + w4;
        a.sc[to] = in ? a.scales[from] : 0;
        if (a.zp) a.zp[to] = in ? a.zeros[from] & 15 : 8;
    }
}

// ---- product ------------------------------------------------------------------------------------------------------------------

// c = a b, or c += a b: a sum that starts does not need zeros in registers
#define NQ_W4_MMA(T)                                                                                                                               \
    if (FIRST)                                                                                                                                     \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"                      \
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));            \
    else                                                                                                                                           \
        asm("mma.sync.aligned.m16n8k16.row.col.f32." T "." T ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"                          \
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))
// (w & MASK) | bits, in one instruction
template <uint32_t MASK>
__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t bits)
{
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w), "n"(MASK), "r"(bits));
    return v;
}
template <class X> struct Operand;
template <> struct Operand<__half> {
    template <bool FIRST>
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        NQ_W4_MMA("f16");
    }
    // what comes off the words of the two rows (z: their zero points, a byte each): 1024 + z, whose last bit is 1, and -(64 + z), whose last bit is 1 / 16
    static __device__ __forceinline__ void zeros(uint32_t z, uint32_t& lo, uint32_t& hi)
    {
        lo = __byte_perm(z, 0x64u, 0x4040);
        hi = __byte_perm(z >> 4, 0xd4u, 0x4040);      // (z's low byte is below 16)
    }
    // A fragment of a step: 0x6400 | n = 1024 + n, 0x6400 | n << 4 = 1024 + 16 n
    static __device__ __forceinline__ void weights(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4])
    {
        const uint32_t w8 = w >> 8, sixteenth = 0x2c002c00u;
        a[0] = masked<0x000f000fu>(w, 0x64006400u);
        a[1] = masked<0x00f000f0u>(w, 0x64006400u);
        a[2] = masked<0x000f000fu>(w8, 0x64006400u);
        a[3] = masked<0x00f000f0u>(w8, 0x64006400u);
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a[0]) : "r"(lo));
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(a[1]) : "r"(sixteenth), "r"(hi));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a[2]) : "r"(lo));
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(a[3]) : "r"(sixteenth), "r"(hi));
    }
};
template <> struct Operand<__nv_bfloat16> {
    template <bool FIRST>
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        NQ_W4_MMA("bf16");
    }
    static __device__ __forceinline__ void zeros(uint32_t z, uint32_t& lo, uint32_t& hi)
    {
        lo = __byte_perm(z, 0x43u, 0x4040);               // 128 + z: seven bits of mantissa hold it
        hi = __byte_perm(z, 0x43u, 0x4141);
    }
    static __device__ __forceinline__ void weights(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            a[i] = masked<0x000f000fu>(w >> (4 * i), 0x43004300u);
            asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(i & 1 ? hi : lo));
        }
    }
};

// the two scales in a word
template <class SC>
__device__ __forceinline__ float2 scales_of(uint32_t w)
{
    if (std::is_same<SC, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// (by 32-bit address: pointers that are moved along lose what space they point to)
__device__ __forceinline__ uint4 load_shared16(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
template <int WORDS>
__device__ __forceinline__ void load_shared(uint32_t at, uint32_t (&v)[WORDS])
{
    if (WORDS == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(at));
    else if (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1 % WORDS]) : "r"(at));
    else asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1 % WORDS]), "=r"(v[2 % WORDS]), "=r"(v[3 % WORDS]) : "r"(at));
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from)
{
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(to), "l"(from), "n"(BYTES) : "memory");
}
template <int LEFT>
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group %0;" :: "n"(LEFT) : "memory"); }
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int GROUPS>
struct W4Unit {
    uint4 w[2];
    uint32_t sc[GROUPS];
    uint32_t zp[(GROUPS + 1) / 2];       // two bytes a group
};
// A warp's units on their way through shared memory, DEPTH of them asked for ahead.  A lane copies the weights that it reads itself; the first lane of
// four copies the scales and zero points of their two rows.
template <int GROUPS, int DEPTH>
struct W4Stream {
    static constexpr int kDepth = DEPTH, kScales = 1024, kZeros = kScales + 32 * GROUPS, kStage = kZeros + 16 * GROUPS, kBytes = kDepth * kStage;
    const char *w, *sc, *zp;             // of the next unit to ask for
    uint32_t place, last;                // of the oldest unit, of the last place
    int at_w, at_sc, at_zp;              // this lane's, in a place
    bool scales;                         // this lane copies them (its zero points: of one group, two bytes, the aligned word that has them)
    __device__ __forceinline__ W4Stream(const char* shared, int lane)
        : place(shared_address(shared)), at_w(lane * 16), at_sc(kScales + (lane >> 2) * 4 * GROUPS), at_zp(kZeros + (lane >> 2) * 2 * GROUPS), scales((lane & 3) == 0)
    {
        last = place + (kDepth - 1) * kStage;
    }
    // goes on with the units from `unit` on
    __device__ __forceinline__ void seek(const W4& a, size_t unit, int lane)
    {
        w = (const char*)a.qw + unit * 1024 + lane * 16;
        sc = (const char*)a.sc + (unit * 8 + (lane >> 2)) * 4 * GROUPS;
        if (a.zp) zp = (const char*)a.zp + unit * 16 * GROUPS + ((lane >> 2) * 2 * GROUPS & ~3);
    }
    // asks for the next unit, into the oldest one's place; without one too: the copies are counted
    __device__ __forceinline__ void ask(bool there, bool zeros)
    {
        if (there)
        {
            copy_async<16>(place + at_w, w);
            copy_async<16>(place + at_w + 512, w + 512);
            if (scales)
            {
                copy_async<4 * GROUPS>(place + at_sc, sc);
                if (zeros) copy_async<GROUPS == 4 ? 8 : 4>(place + (at_zp & ~3), zp);
            }
            w += 1024; sc += 32 * GROUPS;
            if (zeros) zp += 16 * GROUPS;
        }
        copies_end();
        place = place == last ? last - (kDepth - 1) * kStage : place + kStage;
    }
    __device__ __forceinline__ void oldest(W4Unit<GROUPS>& u, bool zeros) const
    {
        copies_done<kDepth - 1>();
        __syncwarp();
        u.w[0] = load_shared16(place + at_w);
        u.w[1] = load_shared16(place + at_w + 512);
        load_shared(place + at_sc, u.sc);
#pragma unroll
        for (int j = 0; j < (GROUPS + 1) / 2; ++j) u.zp[j] = 0x08080808u;
        if (zeros)
        {
            if (GROUPS == 1) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(u.zp[0]) : "r"(place + at_zp));
            else load_shared(place + at_zp, u.zp);
        }
    }
};

// acc += the unit's 16 x 128 weights times rows of x: xs[n] = shared address of the lane's row of tile n at the unit's columns 8 t
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

// shared memory of a CTA
template <int GROUPS, int TILES>
struct W4Plan {
    using Stream = W4Stream<GROUPS, TILES == 4 ? 3 : 4>;
    static constexpr int kPitch = 8 * TILES + 2, kPart = kW4Warps * 16 * kPitch;
    // parts of two items, so that the sums of one wait for the next one's products; of one item where 32 rows leave no room
    static constexpr int kBuffers = TILES == 4 ? 1 : 2;
    static constexpr int kPlanes = kW4Warps * Stream::kBytes, kParts = kBuffers * kPart * 4, kRoom = kW4MaxShared - kPlanes - kParts;      // for rows of x
};

// An item: a block of strips times the rows of one pass over an expert's rows.  Items are in this order: experts, their passes, blocks.
struct W4Cursor {
    int e, pass, block;                  // pass: counted over all experts
    __device__ __forceinline__ void find(const int* s_first, int E)
    {
        int above = E;                   // s_first[e] <= pass < s_first[above], experts without a pass share their successor's
        while (above - e > 1)
        {
            const int m = (e + above) >> 1;
            if (s_first[m] <= pass) e = m;
            else above = m;
        }
    }
    __device__ __forceinline__ void seek(int item, int blocks, const int* s_first, int E)
    {
        pass = item / blocks; block = item % blocks; e = 0;
        find(s_first, E);
    }
    __device__ __forceinline__ void next(int blocks, const int* s_first, int E, int passes)
    {
        if (++block < blocks) return;
        block = 0;
        if (++pass < passes && s_first[e + 1] <= pass) find(s_first, E);
    }
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
#pragma unroll 2
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
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
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
        // two experts a thread; whatever is in start, rows stay inside x and out
        auto at = [&](int e) { return e == 0 ? 0 : min(max(a.start[min(e, a.E)], 0), a.rows); };
        const int e0 = 2 * threadIdx.x, x0 = at(e0), x1 = at(e0 + 1), x2 = at(e0 + 2);
        const int n0 = (max(x1 - x0, 0) + kRows - 1) / kRows, n1 = (max(x2 - x1, 0) + kRows - 1) / kRows;
        const int before = cta_exclusive_sum(n0 + n1, s_warp, passes);
        if (threadIdx.x == 0) { s_first[a.E] = passes; s_row[a.E] = at(a.E); }
        if (e0 < a.E) s_first[e0] = before;
        if (e0 + 1 < a.E) s_first[e0 + 1] = before + n0;
        if (e0 < a.E) s_row[e0] = x0;
        if (e0 + 1 < a.E) s_row[e0 + 1] = x1;
        __syncthreads();
        // rows behind the last expert's
        const int behind = s_row[a.E];
        for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < (size_t)(a.rows - behind) * a.N; i += (size_t)gridDim.x * blockDim.x)
            store_as(a.out, a.out_type, (behind + i / a.N) * a.out_stride + i % a.N, 0.f);
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
    // the planes do not come from a kernel that lets its successors in early: those of a single matrix are asked for before the wait
#pragma unroll 1
    for (int d = 0; d < Stream::kDepth; ++d) ask();
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
            // other rows of x: pieces of 256 columns, in turn to the warps
            pass = now.pass;
            base = s_row[now.e] + (pass - s_first[now.e]) * kRows;
            rows = min(max(s_row[now.e + 1], s_row[now.e]) - base, kRows);
            __syncthreads();
            const int pieces = (c1 - c0 + 1) / 2;
            for (int r = 0, c = warp; r < rows; c += kW4Warps)
            {
                while (c >= pieces) { c -= pieces; ++r; }
                const int k = (c0 + 2 * c) * 128 + lane * 8, there = k < a.K ? 16 : 0;       // zeros behind the last column
                if (r < rows && k < c1 * 128)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(shared_address(s_x) + r * a.pitch + (2 * c * 128 + lane * 8) * 2),
                                 "l"((const X*)a.x + (size_t)(base + r) * a.x_stride + (there ? k : 0)), "r"(there) : "memory");
            }
            copies_end();
            copies_done<0>();                             // (and the units that were asked for before)
            __syncthreads();
        }
        const uint32_t x0 = shared_address(s_x) + (u0 - c0) * 256;
        float acc[TILES][4];
        if (TILES >= 2 && rows <= 8) strip_product<X, SC, GROUPS, 1>(planes, units, zeros, x0, a.pitch, rows, lane, acc, ask);
        else if (TILES == 4 && rows <= 16) strip_product<X, SC, GROUPS, 2>(planes, units, zeros, x0, a.pitch, rows, lane, acc, ask);
        else strip_product<X, SC, GROUPS, TILES>(planes, units, zeros, x0, a.pitch, rows, lane, acc, ask);
        // two buffers: all parts of the item before this one are there, and those of the one before that have been read; one: they have been read
        if (i > i0 || ck > 1) barrier();
        if (Plan::kBuffers == 2 && i > i0) add_up(s_part + ((i - 1) & 1) * Plan::kPart, old_block, old_base, old_rows);
        const uint32_t to = shared_address(s_part + (Plan::kBuffers == 2 ? i & 1 : 0) * Plan::kPart);
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
        if (Plan::kBuffers == 1)
        {
            barrier();
            add_up(s_part, now.block, base, rows);
            if (ck > 1 && i + 1 < i1) cluster_arrive();
        }
        old_block = now.block; old_base = base; old_rows = rows;
        now.next(blocks, s_first, a.E, passes);
    }
    if (Plan::kBuffers == 1) return;
    barrier();
    add_up(s_part + ((i1 - 1) & 1) * Plan::kPart, old_block, old_base, old_rows);
}

bool w4_shape(int E, int N, int K, int g)
{
    return E >= 1 && E <= kW4MaxExperts && N >= 1 && K <= kW4MaxColumns && (g == 32 || g == 64 || g == 128) && K >= g && K % g == 0;
}
int w4_strips(int N) { return (N - 1) / 16 + 1; }
int w4_chunks(int K) { return (K - 1) / 128 + 1; }

// bytes between rows of x in shared memory: 64 off a multiple of 128, so that two rows of a fragment share the banks
int w4_pitch(int C, int ck) { return ((C + ck - 1) / ck) * 256 + 64; }

// clusters of ck CTAs that the device runs at a time, one CTA per SM
template <class K>
int w4_clusters(K* kernel, int ck, int sms, int device, cudaLaunchConfig_t& cfg)
{
    static std::atomic<int> known[16][4];
    if (ck == 1) return sms;
    std::atomic<int>* const at = device < 16 ? &known[device][ck == 2 ? 0 : ck == 4 ? 1 : 2] : nullptr;
    int n = at ? at->load(std::memory_order_relaxed) : 0;
    if (n) return n;
    cfg.gridDim = dim3(ck);
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    if (at) at->store(n, std::memory_order_relaxed);
    return n;
}

// How a matrix is cut: CTAs of a cluster and warps of a CTA that share a strip, both powers of two.  The device takes ceil(blocks / clusters) rounds; a round
// costs a warp its units and what comes per item (measured: sums and barriers as much as a unit and a half, over a cluster three).
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
        const int there = w4_clusters(w4_kernel<X, SC, GROUPS, TILES>, ck, a.sms, device, cfg);
        for (int log_wk = 0; log_wk <= 4 && ck << log_wk <= a.C; ++log_wk)
        {
            const int blocks = (a.S - 1) / (kW4Warps >> log_wk) + 1, units = ((a.C - 1) >> (log_ck + log_wk)) + 1;
            const double cost = (((long long)blocks * experts - 1) / there + 1) * (units + (ck > 1 ? 3.0 : 1.5));
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
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4MaxShared) != cudaSuccess) return fail(NQ_ERR_CUDA, "nq_w4_matmul: shared memory");
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
    const long long most = (long long)a.blocks * (a.start ? a.rows / (8 * TILES) + (a.E < a.rows ? a.E : a.rows) : (a.rows - 1) / (8 * TILES) + 1);
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
    // as many tiles of eight rows as the call has, up to four; fewer where shared memory does not hold that many rows
    const int pitch = w4_pitch(a.C, a.C < 8 ? a.C : 8);
    if (a.rows <= 8 || 16 * pitch > W4Plan<GROUPS, 2>::kRoom) return w4_launch<X, SC, GROUPS, 1>(a, device, st);
    if (a.rows <= 16 || 32 * pitch > W4Plan<GROUPS, 4>::kRoom) return w4_launch<X, SC, GROUPS, 2>(a, device, st);
    return w4_launch<X, SC, GROUPS, 4>(a, device, st);
}
template <class X, class SC>
int w4_groups(const W4& a, int g, int device, cudaStream_t st)
{
    return g == 128 ? w4_tiles<X, SC, 1>(a, device, st) : g == 64 ? w4_tiles<X, SC, 2>(a, device, st) : w4_tiles<X, SC, 4>(a, device, st);
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
    NQ_REQUIRE(q && scales && qw && sc && !zeros == !zp && nq::aligned16(qw) && nq::aligned16(sc), "nq_w4_layout: null or unaligned pointer");
    const int S = nq::w4_strips(N), C = nq::w4_chunks(K);
    NQ_REQUIRE((int64_t)E * S * C <= 0x7fffffff, "nq_w4_layout: too many units");
    nq::w4_layout_kernel<<<(unsigned)((int64_t)E * S * C), 256, 0, (cudaStream_t)stream>>>(
        nq::W4Layout{(const uint8_t*)q, (const uint16_t*)scales, (const uint8_t*)zeros, (uint32_t*)qw, (uint16_t*)sc, (uint8_t*)zp, E, N, K, group, S, C});
    return nq::check_launch("nq_w4_layout");
}

int nq_w4_matmul(const void* x, int type, long long x_stride, const void* qw, const void* sc, int sc_type, const void* zp, const int32_t* start, int rows, int E,
                 int N, int K, int group, void* out, int out_type, long long out_stride, void* stream)
{
    NQ_REQUIRE(nq::w4_shape(E, N, K, group) && rows >= 0, "nq_w4_matmul: rows = %d, E = %d, N = %d, K = %d, group = %d", rows, E, N, K, group);
    NQ_REQUIRE((type == NQ_F16 || type == NQ_BF16) && (sc_type == NQ_F16 || sc_type == NQ_BF16) && (out_type == type || out_type == NQ_F32),
               "nq_w4_matmul: types %d, %d -> %d", type, sc_type, out_type);
    NQ_REQUIRE(start || E == 1, "nq_w4_matmul: %d matrices without the rows' start array", E);
    NQ_REQUIRE(x_stride >= K && out_stride >= N, "nq_w4_matmul: row strides %lld, %lld", x_stride, out_stride);
    if (rows == 0) return NQ_OK;
    NQ_REQUIRE(x && qw && sc && out, "nq_w4_matmul: null pointer");
    NQ_REQUIRE(nq::aligned16(x) && x_stride % 8 == 0 && nq::aligned16(qw) && nq::aligned16(sc), "nq_w4_matmul: rows of x and planes start on 16 bytes");
    nq::W4 a{(const uint4*)qw, (const uint16_t*)sc, (const uint8_t*)zp, x, start, out, x_stride, out_stride, rows, N, K, E, nq::w4_strips(N), nq::w4_chunks(K),
             out_type, 0, 0, 0, 0, 0};
    int device;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&a.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess)
        return nq::fail(NQ_ERR_CUDA, "nq_w4_matmul: no device");
    cudaStream_t st = (cudaStream_t)stream;
    if (type == NQ_F16) return sc_type == NQ_F16 ? nq::w4_groups<__half, __half>(a, group, device, st) : nq::w4_groups<__half, __nv_bfloat16>(a, group, device, st);
    return sc_type == NQ_F16 ? nq::w4_groups<__nv_bfloat16, __half>(a, group, device, st) : nq::w4_groups<__nv_bfloat16, __nv_bfloat16>(a, group, device, st);
}

}  // extern "C"
