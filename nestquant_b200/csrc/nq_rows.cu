// Rows of tokens sorted by expert and back, with the gradients.  pos[t][k] is the place of pick k of token t in the sorted order, a
// permutation of the T topk picks (nq_sort_picks); the places from *live on belong to picks without an expert.
//   dispatch   xs[pos[t][k]] = x[t], zeros for picks without an expert;      its gradient is the sum  dx[t] = sum_k dxs[pos[t][k]]
//   combine    out[t] = sum_k rw[t][k] y[pos[t][k]] over the picks that have an expert;
//              dy[pos[t][k]] = rw[t][k] dout[t] (zeros without an expert), drw[t][k] = <y[pos[t][k]], dout[t]> (0 without one)
// Rows of picks without an expert are never read.  Sums are in 32 bits, in pick order: results do not depend on timing.
//
// All of it is bound by HBM: (1 + topk) rows a token in each direction, read or written once.  Every row is touched in the widest pieces, 16 bytes at most, that
// pointers and strides allow.  In copy and sum a thread has one piece of a token's row and the topk pieces that belong to it, so that
// topk independent loads or stores are in flight per thread (predicated loads: behind branches they went one by one, 80 us instead of 67); the gradient of combine
// has warps per token for the dot products, two, four or eight picks at a time (with places for eight 5,001 x 4 x 1,000 took 11 and 22 us: the registers, and loads
// under predicates that do not hold).  4,096 tokens x 8 picks x 6,144 bf16, us (floor at the copy's 6.54 TB/s): copy 72 (69), sums 66 (69: part of the rows is
// still in L2), combine's gradient 140 (131); 5,001 x 4 x 1,000: 7.5, 8.8, 16.9 (7.7, 7.7, 13.8).  Weighted sums of eight
// 16-bit picks at a time spill 12 bytes of registers, nothing else here spills.
#include <initializer_list>
#include <type_traits>

#include "nq_common.cuh"
#include "nq_types.cuh"

namespace nq {

constexpr int kRowsThreads = 256;

struct Rows {
    const void* src; void* dst;
    const int* pos; const int* live; const void* rw;
    long long src_stride;            // dispatch: elements between the rows of x
    int T, topk, H, rw_type;
    int pieces;                      // of a row
};

// piece i of all tokens' rows: token and piece of its row (a 64-bit division only where there are that many)
__device__ __forceinline__ void piece_of(size_t i, unsigned pieces, size_t& t, unsigned& v)
{
    if (i >> 32) { t = i / pieces; v = (unsigned)(i % pieces); }
    else { t = (unsigned)i / pieces; v = (unsigned)i % pieces; }
}

// a token's row to its picks' places; V = what is copied at a time, src_stride in V
template <class V>
__global__ void __launch_bounds__(kRowsThreads) dispatch_kernel(Rows a)
{
    early_signal();
    grid_dependency_wait();
    const size_t i = (size_t)blockIdx.x * kRowsThreads + threadIdx.x;
    size_t t;
    unsigned v;
    piece_of(i, a.pieces, t, v);
    if (t >= (size_t)a.T) return;
    const V x = ((const V*)a.src)[t * a.src_stride + v];
    const int live = *a.live;
    const int* pos = a.pos + t * a.topk;
    V* dst = (V*)a.dst + v;
#pragma unroll 8
    for (int k = 0; k < a.topk; ++k)
    {
        const int p = pos[k];
        dst[(size_t)p * a.pieces] = p < live ? x : V{};
    }
}

// N elements of a row as floats
template <class T, int N>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[N])
{
    constexpr int kBytes = N * (int)sizeof(T), kStep = kBytes < 16 ? kBytes : 16, kPer = kStep / (int)sizeof(T);
#pragma unroll
    for (int j0 = 0; j0 < N; j0 += kPer)
    {
        union U { typename VecOf<kStep>::type raw; T el[kPer]; __device__ U() {} } u;
        u.raw = *reinterpret_cast<const typename VecOf<kStep>::type*>(p + j0);
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j0 + j] = to_float(u.el[j]);
    }
}
template <class T, int N>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[N])
{
    constexpr int kBytes = N * (int)sizeof(T), kStep = kBytes < 16 ? kBytes : 16, kPer = kStep / (int)sizeof(T);
#pragma unroll
    for (int j0 = 0; j0 < N; j0 += kPer)
    {
        union U { typename VecOf<kStep>::type raw; T el[kPer]; __device__ U() {} } u;
#pragma unroll
        for (int j = 0; j < kPer; ++j) u.el[j] = from_float<T>(v[j0 + j]);
        *reinterpret_cast<typename VecOf<kStep>::type*>(p + j0) = u.raw;
    }
}

// the same as zeros where `there` does not hold: no branch, so that the loads of several picks are on their way together
template <class T, int N>
struct Piece {
    static constexpr int kBytes = N * (int)sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p, bool there)
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
        if (kBytes >= 16)
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t@p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
                             : "+r"(w[i]), "+r"(w[(i + 1) % kWords]), "+r"(w[(i + 2) % kWords]), "+r"(w[(i + 3) % kWords]) : "l"((const char*)p + 4 * i), "r"((unsigned)there) : "memory");
        else if (kBytes == 8)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t@p ld.global.v2.u32 {%0, %1}, [%2];\n\t}" : "+r"(w[0]), "+r"(w[1 % kWords]) : "l"(p), "r"((unsigned)there) : "memory");
        else if (kBytes == 4)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.global.u32 %0, [%1];\n\t}" : "+r"(w[0]) : "l"(p), "r"((unsigned)there) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\t.reg .u16 h;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.u16 h, 0;\n\t@p ld.global.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(w[0]) : "l"(p), "r"((unsigned)there) : "memory");
    }
    __device__ __forceinline__ float at(int j) const
    {
        if (sizeof(T) == 4) return __uint_as_float(w[j % kWords]);
        const unsigned short h = (unsigned short)(w[j / 2 % kWords] >> (16 * (j & 1)));
        if (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(h));
        return __uint_as_float((uint32_t)h << 16);
    }
};

// dst[t] = sum over the token's picks of src[pos] (times rw): dx of dispatch, out of combine
template <class S, class D, int N, int PICKS, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsThreads) sum_kernel(Rows a)
{
    early_signal();
    grid_dependency_wait();
    const size_t i = (size_t)blockIdx.x * kRowsThreads + threadIdx.x;
    size_t t;
    unsigned v;
    piece_of(i, a.pieces, t, v);
    if (t >= (size_t)a.T) return;
    const int live = *a.live;
    const size_t pick = t * a.topk;
    const S* src = (const S*)a.src + (size_t)v * N;
    float sum[N] = {};
    for (int k0 = 0; k0 < a.topk; k0 += PICKS)
    {
        int p[PICKS];
        Piece<S, N> x[PICKS];
#pragma unroll
        for (int k = 0; k < PICKS; ++k) p[k] = k0 + k < a.topk ? a.pos[pick + k0 + k] : 0x7fffffff;
#pragma unroll
        for (int k = 0; k < PICKS; ++k) x[k].load(src + (size_t)p[k] * a.H, p[k] < live);
#pragma unroll
        for (int k = 0; k < PICKS; ++k)
        {
            if (p[k] >= live) continue;
            const float w = WEIGHTED ? load_as(a.rw, a.rw_type, pick + k0 + k) : 1.f;
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += w * x[k].at(j);
        }
    }
    store_piece<D, N>((D*)a.dst + t * a.H + (size_t)v * N, sum);
}

struct CombineBwd {
    const void *dout, *y, *rw; void *dy, *drw;      // dy or drw may be NULL
    const int* pos; const int* live;
    int T, topk, H, rw_type, pieces;
    int warps;                                      // per token: 1, 2, 4 or 8
};

// dy and drw.  Y: type of y and dy, O: of dout, N elements and PICKS picks at a time
template <class Y, class O, int N, int PICKS>
__global__ void __launch_bounds__(kRowsThreads) combine_bwd_kernel(CombineBwd a)
{
    early_signal();
    grid_dependency_wait();
    __shared__ float s_dot[kRowsThreads / 32][PICKS];
    const int per = 32 * a.warps, slot = threadIdx.x / per, r = threadIdx.x % per, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t t = (size_t)blockIdx.x * (kRowsThreads / per) + slot;
    const bool there = t < (size_t)a.T;             // every thread passes the barriers
    const int live = *a.live;
    for (int k0 = 0; k0 < a.topk; k0 += PICKS)
    {
        int p[PICKS];
        float w[PICKS], dot[PICKS] = {};
        const size_t pick = t * a.topk + k0;
        const int n = there ? min(PICKS, a.topk - k0) : 0;
#pragma unroll
        for (int k = 0; k < PICKS; ++k)
        {
            p[k] = k < n ? a.pos[pick + k] : 0;
            w[k] = k < n && p[k] < live ? load_as(a.rw, a.rw_type, pick + k) : 0.f;
        }
        if (there)
            for (unsigned v = r; v < (unsigned)a.pieces; v += per)      // (a row may have 2^31 - 1)
            {
                float d[N];
                Piece<Y, N> y[PICKS];
                if (a.drw)
#pragma unroll
                    for (int k = 0; k < PICKS; ++k) y[k].load((const Y*)a.y + (size_t)p[k] * a.H + (size_t)v * N, k < n && p[k] < live);
                load_piece<O, N>((const O*)a.dout + t * a.H + (size_t)v * N, d);
                if (a.dy)
#pragma unroll
                    for (int k = 0; k < PICKS; ++k)
                    {
                        if (k >= n) continue;
                        float g[N];
#pragma unroll
                        for (int j = 0; j < N; ++j) g[j] = p[k] < live ? w[k] * d[j] : 0.f;
                        store_piece<Y, N>((Y*)a.dy + (size_t)p[k] * a.H + (size_t)v * N, g);
                    }
                if (a.drw)
#pragma unroll
                    for (int k = 0; k < PICKS; ++k)
                        if (k < n && p[k] < live)
#pragma unroll
                            for (int j = 0; j < N; ++j) dot[k] += y[k].at(j) * d[j];
            }
        if (!a.drw) continue;
#pragma unroll
        for (int k = 0; k < PICKS; ++k)
        {
            float s = dot[k];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) s_dot[warp][k] = s;
        }
        if (a.warps == 1) __syncwarp();
        else __syncthreads();
        if (r < n)
        {
            float s = 0.f;
            for (int q = 0; q < a.warps; ++q) s += s_dot[slot * a.warps + q][r];
            store_as(a.drw, a.rw_type, pick + r, s);
        }
        if (a.warps == 1) __syncwarp();
        else __syncthreads();
    }
}

// the most elements, 16 bytes of S at most, that rows of H elements at these pointers can be moved by; a wider type's pieces are stored 16 bytes at a time
template <class S>
int row_step(int H, int widest, std::initializer_list<const void*> ptrs)
{
    int n = 16 / (int)sizeof(S);
    for (; n > 1; n /= 2)
    {
        const size_t align = (size_t)n * widest < 16 ? (size_t)n * widest : 16;
        bool fits = H % n == 0;
        for (const void* p : ptrs) fits = fits && reinterpret_cast<uintptr_t>(p) % align == 0;
        if (fits) break;
    }
    return n;
}
int row_grid(int T, int pieces, unsigned* grid, const char* what)
{
    const size_t ctas = ((size_t)T * pieces + kRowsThreads - 1) / kRowsThreads;
    NQ_REQUIRE(ctas <= 0x7fffffffu, "%s: too many elements", what);
    *grid = (unsigned)ctas;
    return NQ_OK;
}

// picks of a token at a time: a few that a token does not have cost as much as those that it has
template <class F>
void by_picks(int topk, F&& launch)
{
    if (topk <= 2) launch(std::integral_constant<int, 2>());
    else if (topk <= 4) launch(std::integral_constant<int, 4>());
    else launch(std::integral_constant<int, 8>());
}

template <class S, class D, bool WEIGHTED>
int sum_rows(Rows a, cudaStream_t st, const char* what)
{
    const int n = row_step<S>(a.H, (int)(sizeof(D) > sizeof(S) ? sizeof(D) : sizeof(S)), {a.src, a.dst});
    a.pieces = a.H / n;
    unsigned grid;
    if (int e = row_grid(a.T, a.pieces, &grid, what)) return e;
    by_picks(a.topk, [&](auto picks) {
        constexpr int kP = decltype(picks)::value;
        if (n == 8) { if constexpr (sizeof(S) == 2) launch_dependent(sum_kernel<S, D, 8, kP, WEIGHTED>, dim3(grid), dim3(kRowsThreads), 0, st, a); }
        else if (n == 4) launch_dependent(sum_kernel<S, D, 4, kP, WEIGHTED>, dim3(grid), dim3(kRowsThreads), 0, st, a);
        else if (n == 2) launch_dependent(sum_kernel<S, D, 2, kP, WEIGHTED>, dim3(grid), dim3(kRowsThreads), 0, st, a);
        else launch_dependent(sum_kernel<S, D, 1, kP, WEIGHTED>, dim3(grid), dim3(kRowsThreads), 0, st, a);
    });
    return check_launch(what);
}

template <class Y, class O>
int combine_bwd(CombineBwd a, cudaStream_t st)
{
    const int n = row_step<Y>(a.H, (int)(sizeof(O) > sizeof(Y) ? sizeof(O) : sizeof(Y)), {a.dout, a.y, a.dy});
    a.pieces = a.H / n;
    // a warp per token if that makes 64 for each SM; more where there are few tokens and rows are long (3,000 x 6 x 4,096: 67 us, with 16 for each SM 77, eight
    // always 70; 5,001 x 4 x 1,000: 16.9, 17.3, 19.8)
    a.warps = 1;
    while (a.warps < 8 && 32 * a.warps < a.pieces && (long long)a.T * a.warps < 9472) a.warps *= 2;
    const int tokens = kRowsThreads / (32 * a.warps), grid = (a.T - 1) / tokens + 1;
    by_picks(a.topk, [&](auto picks) {
        constexpr int kP = decltype(picks)::value;
        if (n == 8) { if constexpr (sizeof(Y) == 2) launch_dependent(combine_bwd_kernel<Y, O, 8, kP>, dim3(grid), dim3(kRowsThreads), 0, st, a); }
        else if (n == 4) launch_dependent(combine_bwd_kernel<Y, O, 4, kP>, dim3(grid), dim3(kRowsThreads), 0, st, a);
        else if (n == 2) launch_dependent(combine_bwd_kernel<Y, O, 2, kP>, dim3(grid), dim3(kRowsThreads), 0, st, a);
        else launch_dependent(combine_bwd_kernel<Y, O, 1, kP>, dim3(grid), dim3(kRowsThreads), 0, st, a);
    });
    return check_launch("nq_combine_bwd");
}

bool rows_sizes(int type, int T, int topk, int H)
{
    return known_type(type) && T >= 0 && topk >= 1 && H >= 1 && (long long)T * topk <= 0x7fffffffLL;
}

}  // namespace nq

extern "C" {

int nq_dispatch(const void* x, int type, long long row_stride, const int32_t* pos, const int32_t* live, int T, int topk, int H, void* xs, void* stream)
{
    NQ_REQUIRE(nq::rows_sizes(type, T, topk, H) && row_stride >= H, "nq_dispatch: type %d, T = %d, topk = %d, H = %d, row stride %lld", type, T, topk, H, row_stride);
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(x && pos && live && xs, "nq_dispatch: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {x, xs}) && nq::aligned_to(4, {pos, live}), "nq_dispatch: pointers are not aligned to the elements");
    // the widest piece that rows, strides and pointers are whole multiples of
    const size_t size = nq::type_size(type);
    int piece = 16;
    while ((size_t)H * size % piece || (size_t)row_stride * size % piece || reinterpret_cast<uintptr_t>(x) % piece || reinterpret_cast<uintptr_t>(xs) % piece) piece /= 2;
    nq::Rows a{x, xs, pos, live, nullptr, (long long)((size_t)row_stride * size / piece), T, topk, H, 0, (int)((size_t)H * size / piece)};
    unsigned grid;
    if (int e = nq::row_grid(T, a.pieces, &grid, "nq_dispatch")) return e;
    cudaStream_t st = (cudaStream_t)stream;
    if (piece == 16) nq::launch_dependent(nq::dispatch_kernel<uint4>, dim3(grid), dim3(nq::kRowsThreads), 0, st, a);
    else if (piece == 8) nq::launch_dependent(nq::dispatch_kernel<uint2>, dim3(grid), dim3(nq::kRowsThreads), 0, st, a);
    else if (piece == 4) nq::launch_dependent(nq::dispatch_kernel<uint32_t>, dim3(grid), dim3(nq::kRowsThreads), 0, st, a);
    else nq::launch_dependent(nq::dispatch_kernel<uint16_t>, dim3(grid), dim3(nq::kRowsThreads), 0, st, a);
    return nq::check_launch("nq_dispatch");
}

int nq_dispatch_bwd(const void* dxs, int type, const int32_t* pos, const int32_t* live, int T, int topk, int H, void* dx, void* stream)
{
    NQ_REQUIRE(nq::rows_sizes(type, T, topk, H), "nq_dispatch_bwd: type %d, T = %d, topk = %d, H = %d", type, T, topk, H);
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(dxs && pos && live && dx, "nq_dispatch_bwd: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {dxs, dx}) && nq::aligned_to(4, {pos, live}), "nq_dispatch_bwd: pointers are not aligned to the elements");
    nq::Rows a{dxs, dx, pos, live, nullptr, 0, T, topk, H, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (type == NQ_F32) return nq::sum_rows<float, float, false>(a, st, "nq_dispatch_bwd");
    if (type == NQ_F16) return nq::sum_rows<__half, __half, false>(a, st, "nq_dispatch_bwd");
    return nq::sum_rows<__nv_bfloat16, __nv_bfloat16, false>(a, st, "nq_dispatch_bwd");
}

int nq_combine(const void* y, int type, const void* rw, int rw_type, const int32_t* pos, const int32_t* live, int T, int topk, int H, void* out, int out_type,
               void* stream)
{
    NQ_REQUIRE(nq::rows_sizes(type, T, topk, H) && nq::known_type(rw_type) && (out_type == type || out_type == NQ_F32),
               "nq_combine: types %d, %d -> %d, T = %d, topk = %d, H = %d", type, rw_type, out_type, T, topk, H);
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(y && rw && pos && live && out, "nq_combine: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {y}) && nq::aligned_to(nq::type_size(rw_type), {rw}) && nq::aligned_to(4, {pos, live}) &&
               nq::aligned_to(nq::type_size(out_type), {out}), "nq_combine: pointers are not aligned to the elements");
    nq::Rows a{y, out, pos, live, rw, 0, T, topk, H, rw_type, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (type == NQ_F32) return nq::sum_rows<float, float, true>(a, st, "nq_combine");
    if (type == NQ_F16) return out_type == NQ_F32 ? nq::sum_rows<__half, float, true>(a, st, "nq_combine") : nq::sum_rows<__half, __half, true>(a, st, "nq_combine");
    return out_type == NQ_F32 ? nq::sum_rows<__nv_bfloat16, float, true>(a, st, "nq_combine") : nq::sum_rows<__nv_bfloat16, __nv_bfloat16, true>(a, st, "nq_combine");
}

int nq_combine_bwd(const void* dout, int out_type, const void* y, int type, const void* rw, int rw_type, const int32_t* pos, const int32_t* live, int T, int topk,
                   int H, void* dy, void* drw, void* stream)
{
    NQ_REQUIRE(nq::rows_sizes(type, T, topk, H) && nq::known_type(rw_type) && (out_type == type || out_type == NQ_F32),
               "nq_combine_bwd: types %d, %d, %d, T = %d, topk = %d, H = %d", out_type, type, rw_type, T, topk, H);
    if (T == 0 || !(dy || drw)) return NQ_OK;
    NQ_REQUIRE(dout && (y || !drw) && rw && pos && live, "nq_combine_bwd: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {y, dy}) && nq::aligned_to(nq::type_size(rw_type), {rw, drw}) && nq::aligned_to(4, {pos, live}) &&
               nq::aligned_to(nq::type_size(out_type), {dout}), "nq_combine_bwd: pointers are not aligned to the elements");
    nq::CombineBwd a{dout, y, rw, dy, drw, pos, live, T, topk, H, rw_type, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (type == NQ_F32) return nq::combine_bwd<float, float>(a, st);
    if (type == NQ_F16) return out_type == NQ_F32 ? nq::combine_bwd<__half, float>(a, st) : nq::combine_bwd<__half, __half>(a, st);
    return out_type == NQ_F32 ? nq::combine_bwd<__nv_bfloat16, float>(a, st) : nq::combine_bwd<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // extern "C"
