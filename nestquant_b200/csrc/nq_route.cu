// The router's choice and its gradient: logits [T][E] -> expert ids and weights of each token's topk picks.
//
//   choice    by s_e = sigmoid(l_e) + b_e where there is a bias, else by l_e (both scores grow with it): the topk largest, in
//             falling order, equal ones by the lowest id.  Experts whose logit or bias is NaN or -inf are never chosen; where fewer
//             than topk are left, the places behind have id -1 and weight 0, which every kernel of the layer skips.
//   weights   c p_j / sum of the chosen p, or c p_j, with p = sigmoid(l) or p = softmax over all experts.
//             The ratio is formed from p e^(-m), m = min(0, largest chosen logit): no sum underflows, however low the logits are.
//   gradient  (the choice and the bias have none), g = gradient of the weights, r_j = p_j / sum of the chosen p:
//             renormalised sigmoid  dl_j = c r_j (1 - s_j) (g_j - sum_i g_i r_i);  softmax: the same without (1 - s_j);
//             sigmoid as it is      dl_j = c g_j s_j (1 - s_j);   softmax as it is: dl_e = c p_e (g_e - sum_i g_i p_i), g_e = 0 elsewhere.
//
// With a bias the order has to be that of the real numbers, not of their roundings to 32 bits, whose ties would depend on how the
// exponential is computed.  |fp32 score - score| <= 2.7e-7 + 6e-8 |score| with the hardware's exponential and reciprocal: the argument's rounding is off by
// 2^-24 |l|, the power of two by 2^-22 of its value, which the slope s (1 - s) <= min(1/4, e^-|l|) makes 2.2e-8 and 6e-8; the sum rounds by 6e-8 s and
// the reciprocal is off by 1.2e-7 s; the bias adds 6e-8 |score|.  Two neighbours in the sorted list that are
// further apart than 6e-7 + 3e-7 |score| are in the right order, and so are equal logits with equal biases; a row with any other
// neighbours among its first topk + 1 is put in order again in 64 bits (one row of a thousand, with 256 experts).  Where the last pick and
// the one behind it are equal, the pair says nothing of what follows, so the last pick is held against every expert of the row.
//
// A warp per row; lane i holds the experts [i PER, (i + 1) PER), so that the lowest lane that has the largest key also has the lowest id.  The logits are read once
// (floor of 16,384 rows of 256: 2.8 us, and as much for the gradient's zeros); bound by instructions: 14 us with a bias (16 with
// exponential and division as the weights have them), 11 without, gradient 8.6.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "nq_common.cuh"
#include "nq_types.cuh"

namespace nq {

constexpr int kRouteMaxExperts = 1024, kRouteMaxPicks = 32, kRouteWarps = 4;

// order-preserving map of a float to an unsigned; 0 is left for "not eligible"
__device__ __forceinline__ unsigned float_key(float f)
{
    const unsigned u = __float_as_uint(f + 0.f);             // -0 becomes +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_float(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ bool eligible(float f) { return f > -INFINITY; }      // false for NaN
// scores of about this size that are further apart than this are in the right order
__device__ __forceinline__ float in_doubt_below(float score) { return 6e-7f + 3e-7f * fabsf(score); }
__device__ __forceinline__ double exact_score(float l, float b) { return 1.0 / (1.0 + exp(-(double)l)) + (double)b; }
__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
// for the order alone (see above)
__device__ __forceinline__ float quick_sigmoid(float l) { return __fdividef(1.f, 1.f + __expf(-l)); }
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// PER consecutive values of a row from element e0 on; -inf behind the end of the row
template <class L, int PER>
__device__ __forceinline__ void load_run(const L* row, int e0, int E, bool vec, float (&v)[PER])
{
    constexpr int kBytes = PER * (int)sizeof(L), kVec = kBytes < 16 ? kBytes : 16, kPer = kVec / (int)sizeof(L);
    using V = typename VecOf<kVec>::type;
#pragma unroll
    for (int i = 0; i < PER; i += kPer)
    {
        if (vec && e0 + i + kPer <= E)
        {
            union U { V raw; L el[kPer]; __device__ U() {} } u;
            u.raw = *reinterpret_cast<const V*>(row + e0 + i);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i + j] = to_float(u.el[j]);
        }
        else
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i + j] = e0 + i + j < E ? to_float(row[e0 + i + j]) : -INFINITY;
    }
}

// the row's choice again, in 64 bits: pick j goes to lane j
template <class L, int PER>
__device__ __noinline__ int choose_exactly(const L* row, const float* bias, int E, int topk)
{
    const int lane = threadIdx.x & 31;
    double score[PER];
    unsigned left = 0;                                     // experts of this lane that may be chosen
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const int e = lane * PER + i;
        const float l = e < E ? to_float(row[e]) : -INFINITY, b = e < E ? bias[e] : -INFINITY;
        score[i] = exact_score(l, b);
        if (eligible(l) && eligible(b)) left |= 1u << i;
    }
    int mine = -1;
    for (int j = 0; j < topk; ++j)
    {
        double best = 0.0;
        int at = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if ((left >> i & 1) && (at < 0 || score[i] > best)) { best = score[i]; at = i; }
        // the largest, of the lowest lane that has it
        int from = lane;
        bool any = at >= 0;
#pragma unroll
        for (int o = 16; o; o >>= 1)
        {
            const double s = __shfl_xor_sync(0xffffffffu, best, o);
            const int w = __shfl_xor_sync(0xffffffffu, from, o), a = __shfl_xor_sync(0xffffffffu, (int)any, o);
            if (a && (!any || s > best || (s == best && w < from))) { best = s; from = w; any = true; }
        }
        if (!any) break;                                   // warp-uniform: every lane has the same answer
        if (lane == from) left &= ~(1u << at);
        const int e = __shfl_sync(0xffffffffu, lane * PER + at, from);
        if (lane == j) mine = e;
    }
    return mine;
}

// the same among n candidates, one a lane
template <class L>
__device__ __noinline__ int rank_exactly(const L* row, const float* bias, uint2* found, int n, int topk)
{
    const int lane = threadIdx.x & 31, e = lane < n ? (int)found[lane].y : 0;
    const double mine = lane < n ? exact_score(to_float(row[e]), bias[e]) : 0.0;
    int before = 0;
    for (int j = 0; j < n; ++j)
    {
        const double s = __shfl_sync(0xffffffffu, mine, j);
        const int other = __shfl_sync(0xffffffffu, e, j);
        before += s > mine || (s == mine && other < e);
    }
    __syncwarp();
    if (lane < n) found[before].y = e;
    __syncwarp();
    return lane < topk && lane < n ? (int)found[lane].y : -1;
}

template <class L>
__device__ __forceinline__ bool equal_experts(const L* row, const float* bias, int a, int b) { return to_float(row[a]) == to_float(row[b]) && bias[a] == bias[b]; }

// Whether the row's picks have to be ranked again, where a lane's pick and the one behind it (e1) may be in the wrong order (doubt): they are not equal, or
// they are the last pair and an expert of the row is neither equal to the last pick nor apart from it
template <class L>
__device__ __noinline__ bool in_doubt(const L* row, const float* bias, int E, int topk, int my_e, int e1, bool doubt)
{
    if (__any_sync(0xffffffffu, doubt && !equal_experts(row, bias, my_e, e1))) return true;
    const int last = __shfl_sync(0xffffffffu, my_e, topk - 1);
    const float l = to_float(row[last]), b = bias[last], s = quick_sigmoid(l) + b;
    bool any = false;
    for (int e = threadIdx.x & 31; e < E; e += 32)
    {
        const float l1 = to_float(row[e]), b1 = bias[e], s1 = quick_sigmoid(l1) + b1;
        const bool apart = fabsf(s - s1) > in_doubt_below(fmaxf(fabsf(s), fabsf(s1)));
        any |= eligible(l1) && eligible(b1) && !apart && !(l1 == l && b1 == b);
    }
    return __any_sync(0xffffffffu, any);
}

// The `picks` largest keys one by one, whatever they are; pick j to lane j, the last one (picks may be 33) also to next_key, next_e
template <int PER>
__device__ __noinline__ void choose_one_by_one(const unsigned (&keys)[PER], int picks, unsigned& my_key, int& my_e, unsigned& next_key, int& next_e)
{
    const int lane = threadIdx.x & 31;
    unsigned key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = keys[i];
    for (int j = 0; j < picks; ++j)
    {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = max(m, key[i]);
        const unsigned top = __reduce_max_sync(0xffffffffu, m);
        if (!top) break;
        const int from = __ffs(__ballot_sync(0xffffffffu, m == top)) - 1;
        int at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) at = key[i] == top ? i : at;
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = lane == from && i == at ? 0u : key[i];
        const int e = __shfl_sync(0xffffffffu, lane * PER + at, from);
        if (lane == j) { my_key = top; my_e = e; }
        if (j == picks - 1) { next_key = top; next_e = e; }
    }
}

struct Route {
    const void* logits; const float* bias; int64_t* sel; void* rw;
    long long row_stride;
    int T, E, topk, softmax, renorm, rw_type, vec, vec_bias;
    float scale;
};

// weight of the pick that this lane holds (logit l, any = it holds one); denominator: of the softmax over all experts, highest: its largest logit
__device__ __forceinline__ float pick_weight(const Route& a, bool any, float l, float highest, float denominator)
{
    if (a.softmax && !a.renorm) return any ? a.scale * expf(l - highest) / denominator : 0.f;
    if (!a.renorm) return any ? a.scale * sigmoid(l) : 0.f;
    const float high = warp_max(any ? l : -INFINITY);      // (every lane takes part)
    float p = 0.f;
    if (any) p = a.softmax ? expf(l - high) : expf(fminf(l, 0.f) - fminf(high, 0.f)) / (1.f + expf(-fabsf(l)));
    const float sum = warp_sum(p);
    return any ? a.scale * (p / sum) : 0.f;
}

template <class L, int PER>
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(Route a)
{
    early_signal();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (t >= a.T) return;                                  // warp-uniform
    const L* row = (const L*)a.logits + (size_t)t * a.row_stride;
    float v[PER];
    load_run<L, PER>(row, lane * PER, a.E, a.vec, v);
    float highest = 0.f, denominator = 1.f;
    if (a.softmax && !a.renorm)
    {
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = eligible(v[i]) ? fmaxf(m, v[i]) : m;
        highest = warp_max(m);
#pragma unroll
        for (int i = 0; i < PER; ++i) s += eligible(v[i]) ? expf(v[i] - highest) : 0.f;
        denominator = warp_sum(s);
    }
    unsigned key[PER];
    if (a.bias)
    {
        float b[PER];
        load_run<float, PER>(a.bias, lane * PER, a.E, a.vec_bias, b);
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = eligible(v[i]) && eligible(b[i]) ? float_key(quick_sigmoid(v[i]) + b[i]) : 0u;
    }
    else
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = eligible(v[i]) ? float_key(v[i]) : 0u;
    // Pick j to lane j, and behind a biased choice the one that follows it.  No key below the picks-th largest of the lanes' largest keys is among the picks
    // largest, so the few that are not go to the lanes, one each, and count how many are in front of them.  (Taking the largest away pick by pick takes
    // 48 instructions a pick: 16,384 rows of 256 16.5 us without a bias instead of 11.)
    __shared__ uint2 s_found[kRouteWarps][2][34];          // {key, expert}: as found, in order
    uint2 (&found)[2][34] = s_found[threadIdx.x >> 5];
    unsigned my_key = 0, next_key = 0;
    int my_e = -1, next_e = -1;
    const int picks = a.bias ? min(a.topk + 1, a.E) : a.topk;
    unsigned lead = 0, border = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) lead = max(lead, key[i]);
    for (int j = 0; j < picks; ++j)
    {
        const unsigned top = __reduce_max_sync(0xffffffffu, lead);
        border = top;
        if (!top) break;
        lead = lead == top ? 0u : lead;
    }
    border = max(border, 1u);
    if (a.bias && border > 1u)                             // and what may be among them in 64 bits
    {
        const float f = key_float(border), lower = f - in_doubt_below(f);
        border = lower > -INFINITY ? float_key(lower) : 1u;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
    {
        const bool in = key[i] >= border;
        const unsigned m = __ballot_sync(0xffffffffu, in);
        const int at = n + __popc(m & ((1u << lane) - 1u));
        if (in && at < 32) found[0][at] = make_uint2(key[i], lane * PER + i);
        n += __popc(m);
    }
    __syncwarp();
    if (n <= 32 && picks <= 32)
    {
        const uint2 mine = lane < n ? found[0][lane] : make_uint2(0u, 0u);
        int before = 0;
        for (int j = 0; j < n; ++j)
        {
            const uint2 other = found[0][j];
            before += other.x > mine.x || (other.x == mine.x && other.y < mine.y);
        }
        if (lane < n) found[1][before] = mine;
        __syncwarp();
        if (lane < a.topk && lane < n) { my_key = found[1][lane].x; my_e = (int)found[1][lane].y; }
        if (a.topk < picks && a.topk < n) { next_key = found[1][a.topk].x; next_e = (int)found[1][a.topk].y; }
    }
    else
    {
        choose_one_by_one<PER>(key, picks, my_key, my_e, next_key, next_e);
        if (picks == a.topk) next_e = -1;
    }
    if (a.bias)
    {
        // this pick against the one behind it
        unsigned k1 = __shfl_down_sync(0xffffffffu, my_key, 1);
        int e1 = __shfl_down_sync(0xffffffffu, my_e, 1);
        if (lane == a.topk - 1) { k1 = next_key; e1 = next_e; }
        bool doubt = false;
        if (lane < a.topk && my_e >= 0 && e1 >= 0)
        {
            const float s0 = key_float(my_key), s1 = key_float(k1);
            const bool apart = s0 - s1 > in_doubt_below(fmaxf(fabsf(s0), fabsf(s1)));
            if (!apart) doubt = lane == a.topk - 1 || !equal_experts(row, a.bias, my_e, e1);
        }
        if (__any_sync(0xffffffffu, doubt) && in_doubt(row, a.bias, a.E, a.topk, my_e, e1, doubt))
            my_e = n <= 32 && picks <= 32 ? rank_exactly(row, a.bias, found[0], n, a.topk) : choose_exactly<L, PER>(row, a.bias, a.E, a.topk);
    }
    const bool any = lane < a.topk && my_e >= 0;
    const float w = pick_weight(a, any, any ? to_float(row[my_e]) : 0.f, highest, denominator);
    if (lane < a.topk)
    {
        const size_t o = (size_t)t * a.topk + lane;
        a.sel[o] = any ? my_e : -1;
        store_as(a.rw, a.rw_type, o, w);
    }
}

struct RouteBwd {
    const void* logits; const int64_t* sel; const void* drw; void* dlogits;
    long long row_stride;
    int T, E, topk, softmax, renorm, rw_type, vec;
    float scale;
};

template <class L, int PER>
__global__ void __launch_bounds__(32 * kRouteWarps) route_bwd_kernel(RouteBwd a)
{
    early_signal();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (t >= a.T) return;                                  // warp-uniform
    const L* row = (const L*)a.logits + (size_t)t * a.row_stride;
    L* out = (L*)a.dlogits + (size_t)t * a.E;
    float rest[PER];                                       // gradients of the experts that were not chosen
#pragma unroll
    for (int i = 0; i < PER; ++i) rest[i] = 0.f;
    const bool dense = a.softmax && !a.renorm;
    if (!dense) store_run<L, PER>(out, lane * PER, a.E, a.vec, rest);      // (before anything has to be waited for)
    int e = -1;
    float g = 0.f, l = 0.f;
    if (lane < a.topk)
    {
        const size_t o = (size_t)t * a.topk + lane;
        const int64_t id = a.sel[o];
        if (id >= 0 && id < a.E) { e = (int)id; g = load_as(a.drw, a.rw_type, o); l = to_float(row[e]); }
    }
    const bool any = e >= 0;
    float mine = 0.f;                                      // gradient of this lane's pick
    if (a.renorm)
    {
        const float high = warp_max(any ? l : -INFINITY), m = a.softmax ? high : fminf(high, 0.f);
        float p = 0.f;
        if (any) p = a.softmax ? expf(l - m) : expf(fminf(l, 0.f) - m) / (1.f + expf(-fabsf(l)));
        const float sum = warp_sum(p), r = any ? p / sum : 0.f;
        const float mean = warp_sum(g * r);
        mine = a.scale * r * (g - mean) * (a.softmax ? 1.f : 1.f / (1.f + expf(l)));
    }
    else if (!a.softmax) mine = a.scale * g * sigmoid(l) / (1.f + expf(l));
    else
    {
        float v[PER];
        load_run<L, PER>(row, lane * PER, a.E, a.vec, v);
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = eligible(v[i]) ? fmaxf(m, v[i]) : m;
        m = warp_max(m);
#pragma unroll
        for (int i = 0; i < PER; ++i) { v[i] = eligible(v[i]) ? expf(v[i] - m) : 0.f; s += v[i]; }
        s = warp_sum(s);
        if (s == 0.f) s = 1.f;                             // no expert is eligible: every p is 0, as the weights are
        const float p = any ? expf(l - m) / s : 0.f, mean = warp_sum(g * p);
        mine = a.scale * p * (g - mean);
#pragma unroll
        for (int i = 0; i < PER; ++i) rest[i] = -a.scale * (v[i] / s) * mean;
    }
    if (dense) store_run<L, PER>(out, lane * PER, a.E, a.vec, rest);
    __syncwarp();                                          // the chosen experts' values come on top of what other lanes wrote
    if (any) out[e] = from_float<L>(mine);
}

template <template <class, int> class Launch, class A>
int by_width(int type, int E, const A& a, cudaStream_t st)
{
#define NQ_ROUTE_WIDTHS(L)                                  \
    if (E <= 32) Launch<L, 1>::go(a, st);                   \
    else if (E <= 64) Launch<L, 2>::go(a, st);              \
    else if (E <= 128) Launch<L, 4>::go(a, st);             \
    else if (E <= 256) Launch<L, 8>::go(a, st);             \
    else if (E <= 512) Launch<L, 16>::go(a, st);            \
    else Launch<L, 32>::go(a, st)
    if (type == NQ_F32) { NQ_ROUTE_WIDTHS(float); }
    else if (type == NQ_F16) { NQ_ROUTE_WIDTHS(__half); }
    else { NQ_ROUTE_WIDTHS(__nv_bfloat16); }
#undef NQ_ROUTE_WIDTHS
    return 0;
}
template <class L, int PER>
struct RouteLaunch {
    static void go(Route a, cudaStream_t st)
    {
        a.vec = run_aligned<L, PER>(a.logits, a.row_stride);
        a.vec_bias = run_aligned<float, PER>(a.bias, PER);
        launch_dependent(route_kernel<L, PER>, dim3((a.T - 1) / kRouteWarps + 1), dim3(32 * kRouteWarps), 0, st, a);
    }
};
template <class L, int PER>
struct RouteBwdLaunch {
    static void go(RouteBwd a, cudaStream_t st)
    {
        a.vec = run_aligned<L, PER>(a.logits, a.row_stride) && run_aligned<L, PER>(a.dlogits, a.E);
        launch_dependent(route_bwd_kernel<L, PER>, dim3((a.T - 1) / kRouteWarps + 1), dim3(32 * kRouteWarps), 0, st, a);
    }
};

bool route_sizes(int type, int rw_type, int T, int E, int topk, long long row_stride)
{
    return known_type(type) && known_type(rw_type) && T >= 0 && E >= 1 && E <= kRouteMaxExperts && topk >= 1 && topk <= E && topk <= kRouteMaxPicks &&
           row_stride >= E;
}

}  // namespace nq

extern "C" {

int nq_route(const void* logits, int type, long long row_stride, const float* bias, int T, int E, int topk, int score, int renorm, float scale,
             int64_t* sel, void* rw, int rw_type, void* stream)
{
    NQ_REQUIRE(nq::route_sizes(type, rw_type, T, E, topk, row_stride), "nq_route: types %d, %d, T = %d, E = %d (to %d), topk = %d (to %d and E), row stride %lld",
               type, rw_type, T, E, nq::kRouteMaxExperts, topk, nq::kRouteMaxPicks, row_stride);
    NQ_REQUIRE(score == 0 || score == 1, "nq_route: score %d", score);
    NQ_REQUIRE(!(score == 1 && bias), "nq_route: a bias goes with sigmoid scores");
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(logits && sel && rw, "nq_route: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {logits}) && nq::aligned_to(4, {bias}) && nq::aligned_to(8, {sel}) && nq::aligned_to(nq::type_size(rw_type), {rw}),
               "nq_route: pointers are not aligned to the elements");
    nq::by_width<nq::RouteLaunch>(type, E, nq::Route{logits, bias, sel, rw, row_stride, T, E, topk, score, renorm != 0, rw_type, 0, 0, scale}, (cudaStream_t)stream);
    return nq::check_launch("nq_route");
}

int nq_route_bwd(const void* logits, int type, long long row_stride, const int64_t* sel, const void* drw, int rw_type, int T, int E, int topk, int score,
                 int renorm, float scale, void* dlogits, void* stream)
{
    NQ_REQUIRE(nq::route_sizes(type, rw_type, T, E, topk, row_stride), "nq_route_bwd: types %d, %d, T = %d, E = %d (to %d), topk = %d (to %d and E), row stride %lld",
               type, rw_type, T, E, nq::kRouteMaxExperts, topk, nq::kRouteMaxPicks, row_stride);
    NQ_REQUIRE(score == 0 || score == 1, "nq_route_bwd: score %d", score);
    if (T == 0) return NQ_OK;
    NQ_REQUIRE(logits && sel && drw && dlogits, "nq_route_bwd: null pointer");
    NQ_REQUIRE(nq::aligned_to(nq::type_size(type), {logits, dlogits}) && nq::aligned_to(8, {sel}) && nq::aligned_to(nq::type_size(rw_type), {drw}),
               "nq_route_bwd: pointers are not aligned to the elements");
    nq::by_width<nq::RouteBwdLaunch>(type, E, nq::RouteBwd{logits, sel, drw, dlogits, row_stride, T, E, topk, score, renorm != 0, rw_type, 0, scale}, (cudaStream_t)stream);
    return nq::check_launch("nq_route_bwd");
}

}  // extern "C"
