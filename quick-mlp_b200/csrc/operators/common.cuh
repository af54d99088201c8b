// What the kernels of the operators share: element types, 16-byte accesses, reductions over a group of threads.
#pragma once
#include <initializer_list>
#include <type_traits>
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

// VEC consecutive elements as they lie in memory; VEC is 1, 2 or WIDE<T>
template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
// two 16-bit elements at once: one conversion instruction per pair where there is one
__device__ __forceinline__ float2 toPair(const __half* v) { return __half22float2(*reinterpret_cast<const __half2*>(v)); }
__device__ __forceinline__ float2 toPair(const __nv_bfloat16* v)
{
    const uint32_t u = *reinterpret_cast<const uint32_t*>(v);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void fromPair(__half* v, float a, float b) { *reinterpret_cast<__half2*>(v) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void fromPair(__nv_bfloat16* v, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(v) = __floats2bfloat162_rn(a, b); }

template <class T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& p, float (&f)[VEC])
{
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 v = toPair(&p.v[i]);
            f[i] = v.x;
            f[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = Element<T>::to(p.v[i]);
    }
}
template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC])
{
    Pack<T, VEC> p;
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) fromPair(&p.v[i], f[i], f[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.v[i] = Element<T>::from(f[i]);
    }
    return p;
}

// two fp32 operations per instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// an access' elements in pairs (an odd one with a zero)
template <int VEC> constexpr int PAIRS = (VEC + 1) / 2;
template <class T, int VEC>
__device__ __forceinline__ void unpackPairs(const Pack<T, VEC>& p, float2 (&f)[PAIRS<VEC>])
{
    if constexpr (VEC == 1) f[0] = make_float2(Element<T>::to(p.v[0]), 0.f);
    else unpack<T, VEC>(p, *reinterpret_cast<float (*)[VEC]>(&f[0]));
}
template <class T, int VEC>
__device__ __forceinline__ Pack<T, VEC> packPairs(const float2 (&f)[PAIRS<VEC>])
{
    return pack<T, VEC>(*reinterpret_cast<const float (*)[VEC]>(&f[0]));
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

// ---- launches that overlap -----------------------------------------------------------------------------------------------
// Every kernel of the operators is launched so that its launch overlaps the kernel before it (programmatic stream serialisation), and begins with
// chained(), which waits until all kernels before it are complete and their writes visible; what goes in front of the call touches no
// global memory. The gradient of an embedding of a million tokens, five kernels: 111 -> 97 us, of 65536 tokens over 50000 rows, nine: 131 -> 109 us.
// (Kernels that let the next one start while their own last blocks run were slower, 119 and 113 us: its blocks then crowd on the SMs that are free first.)
__device__ __forceinline__ void chained() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... A>
cudaError_t launchChained(void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, int cluster, const A&... arguments)
{
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = block;
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<P>(arguments)...);
}

// ---- mbarriers and bulk copies ---------------------------------------------------------------------------------------
constexpr uint32_t WAIT_LIMIT = 1u << 22;   // polls of an mbarrier before a kernel gives up

__device__ __forceinline__ uint32_t smemAddress(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrierInit(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void barrierInitDone()
{
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ bool barrierTest(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool barrierWait(uint32_t bar, uint32_t parity)
{
    for (uint32_t i = 0; i < WAIT_LIMIT; ++i)
        if (barrierTest(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ void barrierArrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void barrierExpect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// global -> shared, both addresses and the size multiples of 16 bytes; completes on the mbarrier
__device__ __forceinline__ void bulkLoad(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar) : "memory");
}

// whether rows can be read and written 16 bytes at a time
inline bool wide(const Rows& r, int type, int channels)
{
    const int n = 16 / typeBytes(type);
    return r.data == nullptr || ((reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.stride % n == 0 && channels % n == 0);
}

// The access that all of `matrices` allow, as f(integral_constant of elements): 16 bytes, else pairs of elements, else single ones. 672856 tokens of a table of
// 50 bfloat16: forward 37 us in pairs and 70 us one by one, the gradient's sums 36 and 59 us.
template <class T, class F>
cudaError_t byAccess(std::initializer_list<const Rows*> matrices, int type, int channels, F&& f)
{
    bool all = true, pairs = channels % 2 == 0;
    for (const Rows* r : matrices) {
        all = all && wide(*r, type, channels);
        pairs = pairs && (r->data == nullptr || ((reinterpret_cast<uintptr_t>(r->data) % (2 * sizeof(T))) == 0 && r->stride % 2 == 0));
    }
    if (all) return f(std::integral_constant<int, WIDE<T>>());
    if (pairs) return f(std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 1>());
}

// lets a kernel use up to `bytes` of dynamic shared memory on the current device; asked for once per kernel and device
cudaError_t allowShared(const void* kernel, int bytes);

} // namespace ops
} // namespace kernel
} // namespace qmlp
