// Microscaled 4-bit floating point (OCP Microscaling Formats, MXFP4): 32 channels share a power of two, each is an e2m1 number, one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign. The power is floor(log2(largest magnitude)) - 2, at least -127; elements are rounded to the nearest, ties to the
// even code, and 6 is the largest. A block with an infinity or a NaN has the scale 255, which makes all of it NaN.
#pragma once
#include "common.cuh"

namespace qmlp {
namespace kernel {
namespace mx {

using namespace ops;

// exponent + 127 of a block whose largest magnitude has these bits
__device__ __forceinline__ uint32_t scaleOf(uint32_t magnitude)
{
    const uint32_t e = magnitude >> 23;
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^(127 - scale), a normal number for every scale but 255 (zero)
__device__ __forceinline__ float inverseOf(uint32_t scale) { return __uint_as_float(scale == 255 ? 0u : (254 - scale) << 23); }
// 2^(scale - 127)
__device__ __forceinline__ float powerOf(uint32_t scale) { return __uint_as_float(scale == 255 ? 0x7fffffffu : scale == 0 ? 0x00400000u : scale << 23); }

// eight elements, already divided by their scale, to eight codes, the first in the low bits
__device__ __forceinline__ uint32_t encodeEight(const float (&f)[8])
{
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}
// eight codes to their values
__device__ __forceinline__ void decodeEight(uint32_t codes, float (&f)[8])
{
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}

// eight elements of a row from channel c on, zeros behind the last
template <class T>
struct Eight {
    Pack<T, WIDE<T>> v[8 / WIDE<T>];
};
template <class T, bool ALIGNED>
__device__ __forceinline__ Eight<T> loadEight(const T* row, int c, int channels)
{
    Eight<T> r;
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < 8 / WIDE<T>; ++i) r.v[i] = load<T, WIDE<T>>(row + c + i * WIDE<T>);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i / WIDE<T>].v[i % WIDE<T>] = c + i < channels ? row[c + i] : Element<T>::from(0.f);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void unpackEight(const Eight<T>& p, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 8 / WIDE<T>; ++i) unpack<T, WIDE<T>>(p.v[i], *reinterpret_cast<float (*)[WIDE<T>]>(&f[i * WIDE<T>]));
}

// A block of TILE_THREADS threads works on a tile of 128 rows x 128 channels; LANES threads share a row, 8 channels each (16 of them for 128 channels, fewer
// for matrices that are narrower).
constexpr int TILE_THREADS = 256;
template <int LANES> constexpr int TILE_PASSES = MX_TILE * LANES / TILE_THREADS;

// `rows` rows of x from `x` on, channels from 128 * chunk on, to codes (rows of codeBytes) and a tile of scales. `words`: 128 words of shared memory, which
// the caller may use again after its next barrier.
template <class T, int LANES, bool ALIGNED>
__device__ __forceinline__ void quantizeTile(const T* x, long long stride, int rows, int chunk, int channels, unsigned char* codes, int codeBytes, unsigned char* scales,
                                             uint32_t* words)
{
    constexpr int PASSES = TILE_PASSES<LANES>, STEP = TILE_THREADS / LANES;
    const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES, c = chunk * MX_TILE + lane * 8;
    Eight<T> v[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * STEP + first;
        v[i] = {};
        if (r < rows && c < channels) v[i] = loadEight<T, ALIGNED>(x + r * stride, c, channels);
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * STEP + first;
        float f[8];
        unpackEight<T>(v[i], f);
        uint32_t largest = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) largest = max(largest, __float_as_uint(f[j]) & 0x7fffffffu);
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t scale = scaleOf(largest);
        const float inverse = inverseOf(scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = scale == 255 ? 0.f : f[j] * inverse;
        const uint32_t code = encodeEight(f);
        if (r < rows && c / 2 < codeBytes) *reinterpret_cast<uint32_t*>(codes + static_cast<long long>(r) * codeBytes + c / 2) = code;
        uint32_t word = scale << (lane / 4 * 8);
        if constexpr (LANES > 4) word |= __shfl_xor_sync(0xffffffffu, word, 4);
        if constexpr (LANES > 8) word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (lane == 0) words[(r & 31) * 4 + (r >> 5)] = word;
    }
    __syncthreads();
    if (threadIdx.x < MX_TILE_BYTES / 16) *reinterpret_cast<uint4*>(scales + threadIdx.x * 16) = *reinterpret_cast<const uint4*>(words + threadIdx.x * 4);
}
// lanes that a row of `channels` channels takes
inline int lanesOf(int channels) { return channels > 64 ? 16 : channels > 32 ? 8 : 4; }

} // namespace mx
} // namespace kernel
} // namespace qmlp
