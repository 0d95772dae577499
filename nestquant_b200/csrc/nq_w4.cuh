// Products with 4-bit weights that have a scale and a zero point per row and group of 32, 64 or 128 columns:
//   y[r][n] = sum over groups j of s[n][j] sum_{k in j} (q[n][k] - z[n][j]) x[r][k]
// for one matrix, or for one matrix per expert and rows that are sorted by expert.
//
// Layout (nq_w4_layout, once per matrix): units of 16 rows x 128 columns, 1 KB each, unit index (strip C + chunk), as the packed planes of
// the experts.  A unit is eight steps of m16n8k16, weights as A, columns 16 j .. 16 j + 15 in step j; lane (g, t) = (lane / 4, lane % 4) has columns
// 4 t .. 4 t + 3 of each (the operands' k order is free as long as both sides have the same): side by side they are what a 16x256b
// store to tensor memory takes in plain order, so the same planes serve both kernels.  A lane's 32-bit word of a step holds, by nibble: 0, 4 =
// row g, columns 0, 1 of the four; 1, 5 = row g + 8, columns 0, 1; 2, 6 and 3, 7 the same rows, columns 2, 3: each pair is one masked word away from a
// pair of halves.  Word j of lane i sits at ((j / 4) 32 + i) 16 + (j % 4) 4 of the unit.  Scales [unit][g][group of the unit][row g, row g + 8],
// zero points likewise as bytes.  Rows and columns behind the matrix have scale 0.
//
// q - z is exact in fp16 and in bf16 (integers to 15 in magnitude), products and sums of a group are in 32 bits on the tensor pipe, and
// the group's scale is applied to its sum in 32 bits: nothing is rounded to fewer bits before the result.
#pragma once
#include <type_traits>

#include "nq_cluster.cuh"
#include "nq_common.cuh"
#include "nq_scan.cuh"
#include "nq_types.cuh"

namespace nq {

constexpr int kW4Warps = 16, kW4MaxExperts = 1024;
constexpr int kW4MaxShared = 216 * 1024;      // planes, rows of x and partial sums, beside the experts' rows
constexpr int kW4MaxColumns = 32768;          // eight rows of x in a cluster of eight: 66 KB

struct W4 {
    const uint4* qw; const uint16_t* sc; const uint8_t* zp;
    const void* x; const int* start; void* out; int* status;
    long long x_stride, out_stride;
    int rows, N, K, E, S, C, out_type;
    int log_ck, log_wk, pitch, blocks, sms;         // see w4_kernel
    int more, upto;                                 // see w4_other_call
};

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
__device__ __forceinline__ void copy_async_if(bool there, uint32_t to, const void* from)
{
    if (BYTES == 16) asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}" :: "r"(to), "l"(from), "r"((uint32_t)there) : "memory");
    else asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p cp.async.ca.shared.global [%0], [%1], %3;\n\t}" :: "r"(to), "l"(from), "r"((uint32_t)there), "n"(BYTES) : "memory");
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
// STEP: every unit of the strip, or every other one.
template <int GROUPS, int DEPTH, int STEP = 1>
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
        zp = (const char*)a.zp + unit * 16 * GROUPS + ((lane >> 2) * 2 * GROUPS & ~3);
    }
    // Asks for the next unit, into the oldest one's place; without one too: the copies are counted.  (Predicates, not branches: a branch that the compiler
    // cannot prove uniform costs three instructions of its own.)
    __device__ __forceinline__ void ask(bool there, bool zeros)
    {
        copy_async_if<16>(there, place + at_w, w);
        copy_async_if<16>(there, place + at_w + 512, w + 512);
        copy_async_if<4 * GROUPS>(there && scales, place + at_sc, sc);
        if (zeros) copy_async_if<GROUPS == 4 ? 8 : 4>(there && scales, place + (at_zp & ~3), zp);
        w += STEP * 1024; sc += STEP * 32 * GROUPS; zp += STEP * 16 * GROUPS;
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

// The experts' rows and, with ROWS rows a pass, their first passes: row[0 .. E], first[0 .. E] in shared memory; all passes are returned.  Whole CTA,
// kW4MaxExperts / 2 threads at least.  Whatever is in start, rows stay inside x and out: an array that falls anywhere is taken for one of empty experts,
// and the status says so.
template <int ROWS>
__device__ __forceinline__ int expert_passes(const W4& a, int* row, int* first, int* s_warp)
{
    auto at = [&](int e) { return e == 0 ? 0 : min(max(a.start[min(e, a.E)], 0), a.rows); };
    const int e0 = min(2 * (int)threadIdx.x, a.E), x0 = at(e0), x1 = at(e0 + 1), x2 = at(e0 + 2);
    const int n0 = e0 < a.E ? (max(x1 - x0, 0) + ROWS - 1) / ROWS : 0, n1 = e0 + 1 < a.E ? (max(x2 - x1, 0) + ROWS - 1) / ROWS : 0;
    const bool falls = __syncthreads_or(x1 < x0 || x2 < x1);
    int passes;
    const int before = cta_exclusive_sum(falls ? 0 : n0 + n1, s_warp, passes);
    if (threadIdx.x == 0) { first[a.E] = passes; row[a.E] = falls ? 0 : at(a.E); }
    if (e0 < a.E) { first[e0] = before; row[e0] = falls ? 0 : x0; }
    if (e0 + 1 < a.E) { first[e0 + 1] = before + (falls ? 0 : n0); row[e0 + 1] = falls ? 0 : x1; }
    if (falls && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 2;
    __syncthreads();
    return passes;
}
// How many rows the experts have stands in start[E], on the device: `rows` only bounds it, by eight times as much where other ranks have most picks.  Of the launches
// of a call, one for each form that may be the best for it, the one with more < start[E] <= upto does the work; the others end at once.
__device__ __forceinline__ bool w4_other_call(const W4& a)
{
    const int rows = max(a.start[a.E], 0);
    return rows <= a.more || rows > a.upto;
}
// zeros into the rows that no expert has
__device__ __forceinline__ void zero_rows_behind(const W4& a, int behind)
{
    // (in 32 unsigned bits: a step behind 2^31 - 1 is no negative number)
    for (unsigned r = behind + blockIdx.x; r < (unsigned)a.rows; r += gridDim.x)
        for (unsigned n = threadIdx.x; n < (unsigned)a.N; n += blockDim.x) store_as(a.out, a.out_type, (size_t)r * a.out_stride + n, 0.f);
}

}  // namespace nq
