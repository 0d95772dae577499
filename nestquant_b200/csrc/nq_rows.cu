// Rows of tokens sorted by expert and back, with the gradients.  pos[t][k] is the place of pick k of token t in the sorted order, a
// permutation of the T topk picks (nq_sort_picks); the places from *live on belong to picks without an expert.
//   dispatch   xs[pos[t][k]] = x[t], zeros for picks without an expert;      its gradient is the sum  dx[t] = sum_k dxs[pos[t][k]]
//   combine    out[t] = sum_k rw[t][k] y[pos[t][k]] over the picks that have an expert;
//              dy[pos[t][k]] = rw[t][k] dout[t] (zeros without an expert), drw[t][k] = <y[pos[t][k]], dout[t]> (0 without one)
// Rows of picks without an expert are never read.  Sums are in 32 bits, in pick order: results do not depend on timing.
//
// All of it is bound by HBM: (1 + topk) rows a token in each direction, read or written once.  Every row is touched in 16-byte pieces
// where pointers and strides allow it.  In copy and sum a thread has one piece of a token's row and the topk pieces that belong to it, so that
// topk independent loads or stores are in flight per thread; the gradient of combine has whole CTAs or warps per token for the dot
// products, eight picks at a time.
#include <initializer_list>

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

// dst[t] = sum over the token's picks of src[pos] (times rw): dx of dispatch, out of combine
template <class S, class D, int N, bool WEIGHTED>
__global__ void __launch_bounds__(kRowsThreads) sum_kernel(Rows a)
{
    const size_t i = (size_t)blockIdx.x * kRowsThreads + threadIdx.x;
    size_t t;
    unsigned v;
    piece_of(i, a.pieces, t, v);
    if (t >= (size_t)a.T) return;
    const int live = *a.live;
    const size_t pick = t * a.topk;
    const S* src = (const S*)a.src + (size_t)v * N;
    float sum[N] = {};
#pragma unroll 8
    for (int k = 0; k < a.topk; ++k)
    {
        const int p = a.pos[pick + k];
        if (p >= live) continue;
        float x[N];
        load_piece<S, N>(src + (size_t)p * a.H, x);
        const float w = WEIGHTED ? load_as(a.rw, a.rw_type, pick + k) : 1.f;
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += w * x[j];
    }
    store_piece<D, N>((D*)a.dst + t * a.H + (size_t)v * N, sum);
}

struct CombineBwd {
    const void *dout, *y, *rw; void *dy, *drw;      // dy or drw may be NULL
    const int* pos; const int* live;
    int T, topk, H, rw_type, pieces;
    int warps;                                      // per token: 1, 2, 4 or 8
};

// dy and drw.  Y: type of y and dy, O: of dout, N elements at a time
template <class Y, class O, int N>
__global__ void __launch_bounds__(kRowsThreads) combine_bwd_kernel(CombineBwd a)
{
    constexpr int kPicks = 8;
    __shared__ float s_dot[kRowsThreads / 32][kPicks];
    const int per = 32 * a.warps, slot = threadIdx.x / per, r = threadIdx.x % per, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t t = (size_t)blockIdx.x * (kRowsThreads / per) + slot;
    const bool there = t < (size_t)a.T;                   // every thread passes the barriers
    const int live = *a.live;
    for (int k0 = 0; k0 < a.topk; k0 += kPicks)
    {
        int p[kPicks];
        float w[kPicks], dot[kPicks] = {};
        const size_t pick = t * a.topk + k0;
        const int n = there ? min(kPicks, a.topk - k0) : 0;
#pragma unroll
        for (int k = 0; k < kPicks; ++k)
        {
            p[k] = k < n ? a.pos[pick + k] : 0;
            w[k] = k < n && p[k] < live ? load_as(a.rw, a.rw_type, pick + k) : 0.f;
        }
        if (there)
            for (int v = r; v < a.pieces; v += per)
            {
                float d[N];
                load_piece<O, N>((const O*)a.dout + t * a.H + (size_t)v * N, d);
#pragma unroll
                for (int k = 0; k < kPicks; ++k)
                {
                    if (k >= n) continue;
                    const size_t o = (size_t)p[k] * a.H + (size_t)v * N;
                    const bool lives = p[k] < live;
                    if (a.drw && lives)
                    {
                        float y[N];
                        load_piece<Y, N>((const Y*)a.y + o, y);
#pragma unroll
                        for (int j = 0; j < N; ++j) dot[k] += y[j] * d[j];
                    }
                    if (a.dy)
                    {
                        float g[N];
#pragma unroll
                        for (int j = 0; j < N; ++j) g[j] = lives ? w[k] * d[j] : 0.f;
                        store_piece<Y, N>((Y*)a.dy + o, g);
                    }
                }
            }
        if (!a.drw) continue;
#pragma unroll
        for (int k = 0; k < kPicks; ++k)
        {
            float s = dot[k];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) s_dot[warp][k] = s;
        }
        __syncthreads();
        if (r < n)
        {
            float s = 0.f;
            for (int q = 0; q < a.warps; ++q) s += s_dot[slot * a.warps + q][r];
            store_as(a.drw, a.rw_type, pick + r, s);
        }
        __syncthreads();
    }
}

// elements that can be moved at a time: 16 bytes of S if rows and pointers allow it, else one
template <class S>
bool wide_rows(int H, std::initializer_list<const void*> ptrs)
{
    if ((size_t)H * sizeof(S) % 16) return false;
    for (const void* p : ptrs)
        if (!aligned16(p)) return false;
    return true;
}
int row_grid(int T, int pieces, unsigned* grid, const char* what)
{
    const size_t ctas = ((size_t)T * pieces + kRowsThreads - 1) / kRowsThreads;
    NQ_REQUIRE(ctas <= 0x7fffffffu, "%s: too many elements", what);
    *grid = (unsigned)ctas;
    return NQ_OK;
}

template <class S, class D, bool WEIGHTED>
int sum_rows(Rows a, cudaStream_t st, const char* what)
{
    constexpr int kN = 16 / (int)sizeof(S);
    const bool wide = wide_rows<S>(a.H, {a.src, a.dst});
    a.pieces = wide ? a.H / kN : a.H;
    unsigned grid;
    if (int e = row_grid(a.T, a.pieces, &grid, what)) return e;
    if (wide) sum_kernel<S, D, kN, WEIGHTED><<<grid, kRowsThreads, 0, st>>>(a);
    else sum_kernel<S, D, 1, WEIGHTED><<<grid, kRowsThreads, 0, st>>>(a);
    return check_launch(what);
}

template <class Y, class O>
int combine_bwd(CombineBwd a, cudaStream_t st)
{
    constexpr int kN = 16 / (int)sizeof(Y);
    const bool wide = wide_rows<Y>(a.H, {a.dout, a.y, a.dy}) && (size_t)a.H * sizeof(O) % 16 == 0;
    a.pieces = wide ? a.H / kN : a.H;
    a.warps = a.pieces > 128 ? 8 : a.pieces > 64 ? 4 : a.pieces > 32 ? 2 : 1;
    const int tokens = kRowsThreads / (32 * a.warps), grid = (a.T - 1) / tokens + 1;
    if (wide) combine_bwd_kernel<Y, O, kN><<<grid, kRowsThreads, 0, st>>>(a);
    else combine_bwd_kernel<Y, O, 1><<<grid, kRowsThreads, 0, st>>>(a);
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
    // the widest piece that rows, strides and pointers are whole multiples of
    const size_t size = nq::type_size(type);
    int piece = 16;
    while ((size_t)H * size % piece || (size_t)row_stride * size % piece || reinterpret_cast<uintptr_t>(x) % piece || reinterpret_cast<uintptr_t>(xs) % piece) piece /= 2;
    NQ_REQUIRE(piece >= (int)size, "nq_dispatch: pointers are not aligned to the elements");
    nq::Rows a{x, xs, pos, live, nullptr, (long long)((size_t)row_stride * size / piece), T, topk, H, 0, (int)((size_t)H * size / piece)};
    unsigned grid;
    if (int e = nq::row_grid(T, a.pieces, &grid, "nq_dispatch")) return e;
    cudaStream_t st = (cudaStream_t)stream;
    if (piece == 16) nq::dispatch_kernel<uint4><<<grid, nq::kRowsThreads, 0, st>>>(a);
    else if (piece == 8) nq::dispatch_kernel<uint2><<<grid, nq::kRowsThreads, 0, st>>>(a);
    else if (piece == 4) nq::dispatch_kernel<uint32_t><<<grid, nq::kRowsThreads, 0, st>>>(a);
    else nq::dispatch_kernel<uint16_t><<<grid, nq::kRowsThreads, 0, st>>>(a);
    return nq::check_launch("nq_dispatch");
}

int nq_dispatch_bwd(const void* dxs, int type, const int32_t* pos, const int32_t* live, int T, int topk, int H, void* dx, void* stream)
{
    NQ_REQUIRE(nq::rows_sizes(type, T, topk, H), "nq_dispatch_bwd: type %d, T = %d, topk = %d, H = %d", type, T, topk, H);
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(dxs && pos && live && dx, "nq_dispatch_bwd: null pointer");
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
    nq::CombineBwd a{dout, y, rw, dy, drw, pos, live, T, topk, H, rw_type, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (type == NQ_F32) return nq::combine_bwd<float, float>(a, st);
    if (type == NQ_F16) return out_type == NQ_F32 ? nq::combine_bwd<__half, float>(a, st) : nq::combine_bwd<__half, __half>(a, st);
    return out_type == NQ_F32 ? nq::combine_bwd<__nv_bfloat16, float>(a, st) : nq::combine_bwd<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // extern "C"
