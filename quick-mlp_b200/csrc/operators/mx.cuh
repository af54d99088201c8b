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
// a code to its value: an fp32 number with one bit of mantissa, whose exponent is off by 126
__device__ __forceinline__ float decodeOne(uint32_t code) { return __uint_as_float((code & 7) << 22 | (code & 8) << 28) * 0x1p126f; }
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

// SIXTEEN channels of a row as they lie in memory; ALIGNED: by accesses of 16 bytes, else one by one
constexpr int SIXTEEN = 16;
template <class T>
struct Sixteen {
    Pack<T, WIDE<T>> v[SIXTEEN / WIDE<T>];
};
// of which `left` (at least one) are there. Asked for unconditionally, what is not there as the first again: a load that depends on a condition is waited for
// where it is issued (131072 rows of 1024 bfloat16 quantised in 83 us, without conditions in 57). trim() makes zeros of what is not there.
// ONCE: read by no other thread, and not to displace the codes in L2 (16384 rows of 4096: 26.8 us, so 23.6).
template <class T, bool ALIGNED, bool ONCE = false>
__device__ __forceinline__ Sixteen<T> loadSixteen(const T* at, int left)
{
    Sixteen<T> r;
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < SIXTEEN / WIDE<T>; ++i) {
            const uint4* from = reinterpret_cast<const uint4*>(at + (i * WIDE<T> < left ? i * WIDE<T> : 0));
            const uint4 u = ONCE ? __ldcs(from) : *from;
            memcpy(&r.v[i], &u, sizeof(u));
        }
    } else {
#pragma unroll
        for (int i = 0; i < SIXTEEN; ++i) r.v[i / WIDE<T>].v[i % WIDE<T>] = at[i < left ? i : 0];
    }
    return r;
}
template <class T, bool ALIGNED>
__device__ __forceinline__ void trim(Sixteen<T>& v, int left)
{
    if (left >= SIXTEEN) return;
    constexpr int STEP = ALIGNED ? WIDE<T> : 1;
#pragma unroll
    for (int i = 0; i < SIXTEEN; i += STEP)
        if (i >= left) {
#pragma unroll
            for (int j = 0; j < STEP; ++j) v.v[i / WIDE<T>].v[(i + j) % WIDE<T>] = Element<T>::from(0.f);
        }
}
// bits of the largest magnitude as fp32, a NaN's if there is one; 16-bit elements are compared in pairs
template <class T>
__device__ __forceinline__ uint32_t largestOf(const Sixteen<T>& p)
{
    if constexpr (std::is_same<T, float>::value) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < SIXTEEN; ++i) m = max(m, __float_as_uint(p.v[i / WIDE<T>].v[i % WIDE<T>]) & 0x7fffffffu);
        return m;
    } else {
        using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        Pair m[4];
        Pair w[SIXTEEN / 2];
        memcpy(w, &p, sizeof(w));
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = __hmax2_nan(__habs2(w[i]), __habs2(w[i + 4]));
        m[0] = __hmax2_nan(__hmax2_nan(m[0], m[1]), __hmax2_nan(m[2], m[3]));
        return __float_as_uint(Element<T>::to(__hmax_nan(m[0].x, m[0].y))) & 0x7fffffffu;
    }
}
// codes of sixteen elements whose block has this scale
template <class T>
__device__ __forceinline__ uint2 encodeSixteen(const Sixteen<T>& p, uint32_t scale)
{
    float f[SIXTEEN];
    const float inverse = inverseOf(scale);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        // (a power of two that bfloat16 has: products of pairs are exact, or too small to matter)
        const __nv_bfloat162 pair = __float2bfloat162_rn(inverse);
        __nv_bfloat162 w[SIXTEEN / 2];
        memcpy(w, &p, sizeof(w));
#pragma unroll
        for (int i = 0; i < SIXTEEN / 2; ++i) {
            w[i] = __hmul2(w[i], pair);
            f[2 * i] = __low2float(w[i]);
            f[2 * i + 1] = __high2float(w[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < SIXTEEN / WIDE<T>; ++i) unpack<T, WIDE<T>>(p.v[i], *reinterpret_cast<float (*)[WIDE<T>]>(&f[i * WIDE<T>]));
#pragma unroll
        for (int i = 0; i < SIXTEEN; ++i) f[i] *= inverse;
    }
    uint2 r = {encodeEight(*reinterpret_cast<const float (*)[8]>(&f[0])), encodeEight(*reinterpret_cast<const float (*)[8]>(&f[8]))};
    if (scale == 255) r = make_uint2(0, 0);
    return r;
}

// A block of TILE_THREADS threads works on a tile of 128 rows x 128 channels. LANES threads share a row, 16 channels each (8 of them for 128 channels,
// fewer for matrices that are narrower), two neighbours a block of 32. Rows that 16-byte accesses cannot read go through shared memory, read side by side (20011
// rows of 777 floats: 27 us with 16 elements of a row per thread, which meet the same sectors 16 times; 46 us with a warp per row and its maximum by redux; 23 us so).
constexpr int TILE_THREADS = 256, TILE_WARPS = TILE_THREADS / 32;

// `rows` rows of x, channels from 128 * chunk on, to codes (rows of codeBytes) and a tile of scales; tileScales: 512 bytes of shared memory.
template <class T, int LANES, bool ALIGNED>
__device__ __forceinline__ void quantizeTile(const T* x, long long stride, int rows, int chunk, int channels, unsigned char* codes, int codeBytes, unsigned char* scales,
                                             unsigned char* tileScales)
{
    if constexpr (LANES < 8 || !ALIGNED) {   // the blocks and rows that are not there
        if (threadIdx.x < MX_TILE) *reinterpret_cast<uint32_t*>(tileScales + threadIdx.x * 4) = 0;
        __syncthreads();
    }
    if constexpr (ALIGNED) {
        constexpr int PASSES = MX_TILE * LANES / TILE_THREADS, STEP = TILE_THREADS / LANES;
        const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES, c = chunk * MX_TILE + lane * SIXTEEN, left = channels - c;
        const T* from = x + (left > 0 ? c : 0);
        Sixteen<T> v[PASSES];
#pragma unroll
        for (int i = 0; i < PASSES; ++i) v[i] = loadSixteen<T, true, true>(from + min(i * STEP + first, rows - 1) * stride, left);
        unsigned char* to = codes + static_cast<long long>(first) * codeBytes + c / 2;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = i * STEP + first;
            trim<T, true>(v[i], r < rows ? left : 0);
            uint32_t largest = largestOf<T>(v[i]);
            largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            const uint32_t scale = scaleOf(largest);
            const uint2 code = encodeSixteen<T>(v[i], scale);
            if (r < rows && c / 2 < codeBytes) *reinterpret_cast<uint2*>(to) = code;
            to += STEP * codeBytes;
            if ((lane & 1) == 0) tileScales[(r & 31) * 16 + (r >> 5) * 4 + lane / 2] = static_cast<unsigned char>(scale);
        }
    } else {
        // through shared memory: 32 rows at a time, read side by side, taken up again 16 channels a thread
        constexpr int CHANNELS = LANES * SIXTEEN, ROWS = TILE_THREADS / LANES, PER = ROWS * CHANNELS / TILE_THREADS, PITCH = CHANNELS + 16 / static_cast<int>(sizeof(T));
        __shared__ __align__(16) T staged[ROWS * PITCH];
        const int lane = threadIdx.x % LANES, mine = threadIdx.x / LANES, c = chunk * MX_TILE + lane * SIXTEEN, left = channels - c;
        const int column = threadIdx.x % CHANNELS, line = threadIdx.x / CHANNELS, channel = min(chunk * MX_TILE + column, channels - 1);
        constexpr int LINES = TILE_THREADS / CHANNELS;
        T v[PER];
        const T* from = x + channel;
        auto ask = [&](int begin) {
            if (begin + ROWS <= rows) {
                const T* row = from + (begin + line) * stride;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    v[i] = *row;
                    row += LINES * stride;
                }
            } else {
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] = from[min(begin + i * LINES + line, rows - 1) * stride];
            }
        };
        ask(0);
        for (int begin = 0; begin < rows; begin += ROWS) {
#pragma unroll
            for (int i = 0; i < PER; ++i) staged[(i * LINES + line) * PITCH + column] = v[i];
            __syncthreads();
            ask(begin + ROWS);
            const int r = begin + mine;
            Sixteen<T> part;
#pragma unroll
            for (int i = 0; i < SIXTEEN / WIDE<T>; ++i) part.v[i] = load<T, WIDE<T>>(&staged[mine * PITCH + lane * SIXTEEN + i * WIDE<T>]);
            trim<T, false>(part, r < rows ? left : 0);
            uint32_t largest = largestOf<T>(part);
            largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            const uint32_t scale = scaleOf(largest);
            const uint2 code = encodeSixteen<T>(part, scale);
            if (r < rows && c / 2 < codeBytes) *reinterpret_cast<uint2*>(codes + static_cast<long long>(r) * codeBytes + c / 2) = code;
            if (r < MX_TILE && (lane & 1) == 0) tileScales[(r & 31) * 16 + (r >> 5) * 4 + lane / 2] = static_cast<unsigned char>(scale);
            __syncthreads();
        }
    }
    __syncthreads();
    if (threadIdx.x < MX_TILE_BYTES / 16) *reinterpret_cast<uint4*>(scales + threadIdx.x * 16) = *reinterpret_cast<const uint4*>(tileScales + threadIdx.x * 16);
}
// calls f(integral_constant of LANES, of ALIGNED) for rows of `channels` elements of `type`
template <class F>
cudaError_t byLanes(const Rows& rows, int type, int channels, F&& f)
{
    auto aligned = [&](auto lanes) { return wide(rows, type, channels) ? f(lanes, std::true_type()) : f(lanes, std::false_type()); };
    if (channels > 64) return aligned(std::integral_constant<int, 8>());
    if (channels > 32) return aligned(std::integral_constant<int, 4>());
    return aligned(std::integral_constant<int, 2>());
}

} // namespace mx
} // namespace kernel
} // namespace qmlp
