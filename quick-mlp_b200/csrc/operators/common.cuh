// What the kernels of the operators share: element types, 16-byte accesses, reductions over a group of threads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "operators.h"

namespace qmlp {
namespace kernel {
namespace ops {

template <class T> struct Element;
template <> struct Element<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct Element<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct Element<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// elements of a 16-byte access
template <class T> constexpr int WIDE = 16 / static_cast<int>(sizeof(T));

// VEC consecutive elements as they lie in memory; VEC is 1 or WIDE<T>
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&f)[VEC])
{
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = Element<T>::to(p.v[i]);
}
template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC])
{
    Pack<T, VEC> p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.v[i] = Element<T>::from(f[i]);
    return p;
}
// 16-byte accesses go through uint4, so that they stay one instruction
template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load(const T* at)
{
    if constexpr (sizeof(T) * VEC == 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(at);
        return *reinterpret_cast<const Pack<T, VEC>*>(&u);
    } else {
        return *reinterpret_cast<const Pack<T, VEC>*>(at);
    }
}
template <class T, int VEC>
__device__ __forceinline__ void store(T* at, const Pack<T, VEC>& p)
{
    if constexpr (sizeof(T) * VEC == 16) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(&p);
    else *reinterpret_cast<Pack<T, VEC>*>(at) = p;
}

// an element of a vector whose type is known at run time (parameters: float32 or the features' type)
__device__ __forceinline__ float element(const Vector& v, long long i)
{
    switch (v.type) {
    case TYPE_FLOAT: return static_cast<const float*>(v.data)[i];
    case TYPE_HALF: return __half2float(static_cast<const __half*>(v.data)[i]);
    default: return __bfloat162float(static_cast<const __nv_bfloat16*>(v.data)[i]);
    }
}
__device__ __forceinline__ void storeElement(void* data, int type, long long i, float f)
{
    switch (type) {
    case TYPE_FLOAT: static_cast<float*>(data)[i] = f; break;
    case TYPE_HALF: static_cast<__half*>(data)[i] = __float2half_rn(f); break;
    default: static_cast<__nv_bfloat16*>(data)[i] = __float2bfloat16_rn(f); break;
    }
}

// sum over the G lanes (a power of two, at most 32) that share a row
template <int G>
__device__ __forceinline__ float groupSum(float v)
{
#pragma unroll
    for (int o = G / 2; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// whether rows can be read and written 16 bytes at a time
inline bool wide(const Rows& r, int type, int channels)
{
    const int n = 16 / typeBytes(type);
    return r.data == nullptr || ((reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.stride % n == 0 && channels % n == 0);
}

} // namespace ops
} // namespace kernel
} // namespace qmlp
