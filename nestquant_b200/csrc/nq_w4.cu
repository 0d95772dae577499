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
#include "nq_common.cuh"
#include "nq_types.cuh"

namespace nq {

constexpr int kW4Warps = 8, kW4Tiles = 4, kW4Rows = 8 * kW4Tiles;       // rows of x in a pass

struct W4 {
    const uint4* qw; const uint16_t* sc; const uint8_t* zp;
    const void* x; const int* start; void* out;
    long long x_stride, out_stride;
    int rows, N, K, E, S, C, out_type, sc_bf16;
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

template <class X> struct Operand;
template <> struct Operand<__half> {
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // what is subtracted from the words of the two rows: 1024 + z and 64 + z
    static __device__ __forceinline__ void zeros(int z0, int z1, uint32_t& lo, uint32_t& hi)
    {
        const __half2 a = __half2half2(__int2half_rn(1024 + z0)), b = __half2half2(__int2half_rn(-64 - z1));
        lo = *reinterpret_cast<const uint32_t*>(&a); hi = *reinterpret_cast<const uint32_t*>(&b);
    }
    // A fragment of a step: 0x6400 | n = 1024 + n, 0x6400 | n << 4 = 1024 + 16 n
    static __device__ __forceinline__ void weights(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4])
    {
        const uint32_t w8 = w >> 8, sixteenth = 0x2c002c00u;
        a[0] = (w & 0x000f000fu) | 0x64006400u;
        a[1] = (w & 0x00f000f0u) | 0x64006400u;
        a[2] = (w8 & 0x000f000fu) | 0x64006400u;
        a[3] = (w8 & 0x00f000f0u) | 0x64006400u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a[0]) : "r"(lo));
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(a[1]) : "r"(sixteenth), "r"(hi));
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(a[2]) : "r"(lo));
        asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(a[3]) : "r"(sixteenth), "r"(hi));
    }
};
template <> struct Operand<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void zeros(int z0, int z1, uint32_t& lo, uint32_t& hi)
    {
        lo = (0x4300u | z0) * 0x10001u;                   // 128 + z: seven bits of mantissa hold it
        hi = (0x4300u | z1) * 0x10001u;
    }
    static __device__ __forceinline__ void weights(uint32_t w, uint32_t lo, uint32_t hi, uint32_t (&a)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            a[i] = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            asm("sub.rn.bf16x2 %0, %0, %1;" : "+r"(a[i]) : "r"(i & 1 ? hi : lo));
        }
    }
};

__device__ __forceinline__ float scale_of(uint32_t bits, bool bf16)
{
    return bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}

// a strip of 16 rows of one expert's matrix per CTA, the units of its rows split over the warps.  GROUPS: of a unit (1, 2, 4)
template <class X, int GROUPS>
__global__ void __launch_bounds__(32 * kW4Warps) w4_kernel(W4 a)
{
    __shared__ float s_part[kW4Warps][kW4Rows][17];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int strip = blockIdx.x, e = blockIdx.y;
    int r0 = 0, r1 = a.rows;
    if (a.start)
    {
        // (whatever is in start, rows stay inside x and out)
        r0 = e == 0 ? 0 : min(max(a.start[e], 0), a.rows);
        r1 = e == a.E ? a.rows : min(max(a.start[e + 1], r0), a.rows);
    }
    if (e == a.E)
    {
        // rows behind the last expert's
        for (int i = threadIdx.x; i < (r1 - r0) * 16; i += blockDim.x)
            if (strip * 16 + i % 16 < a.N) store_as(a.out, a.out_type, (size_t)(r0 + i / 16) * a.out_stride + strip * 16 + i % 16, 0.f);
        return;
    }
    const size_t unit0 = ((size_t)e * a.S + strip) * a.C;
    for (int base = r0; base < r1; base += kW4Rows)
    {
        float acc[kW4Tiles][4] = {};
        for (int c = warp; c < a.C; c += kW4Warps)
        {
            const size_t unit = unit0 + c;
            uint4 w[2];
            w[0] = a.qw[unit * 64 + lane];
            w[1] = a.qw[unit * 64 + 32 + lane];
            const uint32_t* words = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
            for (int j = 0; j < GROUPS; ++j)
            {
                const size_t at = unit * 16 * GROUPS + (g * GROUPS + j) * 2;
                const uint32_t s2 = *reinterpret_cast<const uint32_t*>(a.sc + at);
                int z0 = 8, z1 = 8;
                if (a.zp) { z0 = a.zp[at]; z1 = a.zp[at + 1]; }
                uint32_t lo, hi;
                Operand<X>::zeros(z0, z1, lo, hi);
                float part[kW4Tiles][4] = {};
#pragma unroll
                for (int q = 0; q < 4 / GROUPS; ++q)
                {
                    const int G = j * (4 / GROUPS) + q, k = c * 128 + G * 32 + 8 * t;
                    uint32_t a0[4], a1[4];
                    Operand<X>::weights(words[2 * G], lo, hi, a0);
                    Operand<X>::weights(words[2 * G + 1], lo, hi, a1);
#pragma unroll
                    for (int n = 0; n < kW4Tiles; ++n)
                    {
                        const int r = base + 8 * n + g;
                        uint4 b = {};
                        if (r < r1 && k < a.K) b = *reinterpret_cast<const uint4*>((const X*)a.x + r * a.x_stride + k);
                        Operand<X>::mma(part[n], a0, b.x, b.y);
                        Operand<X>::mma(part[n], a1, b.z, b.w);
                    }
                }
                const float s0 = scale_of(s2 & 0xffffu, a.sc_bf16), s1 = scale_of(s2 >> 16, a.sc_bf16);
#pragma unroll
                for (int n = 0; n < kW4Tiles; ++n)
                {
                    acc[n][0] += s0 * part[n][0]; acc[n][1] += s0 * part[n][1];
                    acc[n][2] += s1 * part[n][2]; acc[n][3] += s1 * part[n][3];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kW4Tiles; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_part[warp][8 * n + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[n][i];
        __syncthreads();
        for (int i = threadIdx.x; i < kW4Rows * 16; i += blockDim.x)
        {
            const int r = i / 16, n = i % 16;
            if (base + r < r1 && strip * 16 + n < a.N)
            {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kW4Warps; ++w) sum += s_part[w][r][n];
                store_as(a.out, a.out_type, (size_t)(base + r) * a.out_stride + strip * 16 + n, sum);
            }
        }
        __syncthreads();
    }
}

bool w4_shape(int E, int N, int K, int g)
{
    return E >= 1 && E <= 65534 && N >= 1 && (g == 32 || g == 64 || g == 128) && K >= g && K % g == 0;
}
int w4_strips(int N) { return (N - 1) / 16 + 1; }
int w4_chunks(int K) { return (K - 1) / 128 + 1; }

template <class X>
void w4_launch(const W4& a, int g, dim3 grid, cudaStream_t st)
{
    if (g == 128) w4_kernel<X, 1><<<grid, 32 * kW4Warps, 0, st>>>(a);
    else if (g == 64) w4_kernel<X, 2><<<grid, 32 * kW4Warps, 0, st>>>(a);
    else w4_kernel<X, 4><<<grid, 32 * kW4Warps, 0, st>>>(a);
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
             out_type, sc_type == NQ_BF16};
    const dim3 grid(a.S, start ? E + 1 : 1);
    if (type == NQ_F16) nq::w4_launch<__half>(a, group, grid, (cudaStream_t)stream);
    else nq::w4_launch<__nv_bfloat16>(a, group, grid, (cudaStream_t)stream);
    return nq::check_launch("nq_w4_matmul");
}

}  // extern "C"
