// Element types of the operators around the routed experts (NQ_F32, NQ_F16, NQ_BF16): conversions, whole vectors, alignment.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "nq_common.cuh"

namespace nq {

inline bool known_type(int t) { return t == NQ_F32 || t == NQ_F16 || t == NQ_BF16; }
inline int type_size(int t) { return t == NQ_F32 ? 4 : 2; }

template <int BYTES> struct VecOf;
template <> struct VecOf<2> { using type = uint16_t; };
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<8> { using type = uint2; };
template <> struct VecOf<16> { using type = uint4; };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// scalars whose type is known at run time only
__device__ __forceinline__ float load_as(const void* p, int type, size_t i)
{
    return type == NQ_F32 ? ((const float*)p)[i] : type == NQ_F16 ? __half2float(((const __half*)p)[i]) : __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int type, size_t i, float v)
{
    if (type == NQ_F32) ((float*)p)[i] = v;
    else if (type == NQ_F16) ((__half*)p)[i] = __float2half_rn(v);
    else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}

// whether rows of this stride (in elements) can be read in runs of PER elements, 16 bytes at most at a time
template <class T, int PER>
inline bool run_aligned(const void* p, long long row_stride)
{
    const int bytes = PER * (int)sizeof(T), v = bytes < 16 ? bytes : 16;
    return reinterpret_cast<uintptr_t>(p) % v == 0 && row_stride * (long long)sizeof(T) % v == 0;
}

// PER consecutive values of a row of E
template <class T, int PER>
__device__ __forceinline__ void store_run(T* row, int e0, int E, bool vec, const float (&v)[PER])
{
    constexpr int kBytes = PER * (int)sizeof(T), kVec = kBytes < 16 ? kBytes : 16, kPer = kVec / (int)sizeof(T);
    using V = typename VecOf<kVec>::type;
#pragma unroll
    for (int i = 0; i < PER; i += kPer)
    {
        if (vec && e0 + i + kPer <= E)
        {
            union U { V raw; T el[kPer]; __device__ U() {} } u;
#pragma unroll
            for (int j = 0; j < kPer; ++j) u.el[j] = from_float<T>(v[i + j]);
            *reinterpret_cast<V*>(row + e0 + i) = u.raw;
        }
        else
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (e0 + i + j < E) row[e0 + i + j] = from_float<T>(v[i + j]);
    }
}

}  // namespace nq
