// Dropout: y_i = residual_i + [u_i >= T] x_i 65536 / (65536 - T) over the elements i of (rows, channels), in the order of the rows. T is the probability in
// units of 2^-16, so that the expected value is x_i exactly. The u_i are 16-bit numbers of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random
// numbers: as easy as 1, 2, 3, SC 2011): the key is the seed, the counter (i div 8, offset + step), and each of its four words gives two elements, the low
// half first. Nothing but seed and offset has to be kept: the gradient is the same kernel on dy, without a residual. The numbers depend on an element's
// place among the elements, not on strides or on how the kernel splits its work.
//
// A thread takes groups of 8 elements, one generator call each. Bound by memory, with a third of the machine's instructions left: 32768 rows of 4096 bfloat16 forward with a
// residual and the gradient 233 us (5.8 TB/s); 1000003 rows of 64 half 41 us either way (6.2 TB/s; 49 us with loads that depend on a condition and keys added up).
// Rows that are neither dense nor apart by 16 bytes go element by element, at a quarter of the rate: 32768 rows of 4095 half, 4096 apart, 344 us, dense 86.
#include "common.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

constexpr int THREADS = 256, GROUP = 8;

// how rows lie: one behind the other; 8 elements of a row per access; whatever else
enum Access : int { FLAT = 0, ROWS = 1, SINGLE = 2 };

// what all elements share: the rounds' keys, which go from the kernel's arguments straight into its instructions (added up per call they were 20 of 122
// instructions for 8 elements)
struct Numbers {
    uint32_t low[10], high[10];
    uint32_t cut;   // T << 16
    float scale;
};
// the four words of a counter
__device__ __forceinline__ void philox(unsigned long long group, unsigned long long offset, const Numbers& keys, uint32_t (&c)[4])
{
    c[0] = static_cast<uint32_t>(group);
    c[1] = static_cast<uint32_t>(group >> 32);
    c[2] = static_cast<uint32_t>(offset);
    c[3] = static_cast<uint32_t>(offset >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const unsigned long long a = 0xD2511F53ull * c[0], b = 0xCD9E8D57ull * c[2];
        c[0] = static_cast<uint32_t>(b >> 32) ^ c[1] ^ keys.low[round];
        c[1] = static_cast<uint32_t>(b);
        c[2] = static_cast<uint32_t>(a >> 32) ^ c[3] ^ keys.high[round];
        c[3] = static_cast<uint32_t>(a);
    }
}
// whether element j of a group is kept: its 16 bits are compared where they lie, or shifted to the upper half
__device__ __forceinline__ bool kept(const uint32_t (&word)[4], int j, uint32_t cut) { return (j & 1 ? word[j / 2] : word[j / 2] << 16) >= cut; }

template <class T>
struct Eight {
    Pack<T, WIDE<T>> v[GROUP / WIDE<T>];
};
template <class T>
__device__ __forceinline__ Eight<T> loadEight(const T* at)
{
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < GROUP / WIDE<T>; ++i) r.v[i] = load<T, WIDE<T>>(at + i * WIDE<T>);
    return r;
}
template <class T>
__device__ __forceinline__ void unpackEight(const Eight<T>& p, float (&f)[GROUP])
{
#pragma unroll
    for (int i = 0; i < GROUP / WIDE<T>; ++i) unpack<T, WIDE<T>>(p.v[i], *reinterpret_cast<float (*)[WIDE<T>]>(&f[i * WIDE<T>]));
}

template <class T, int ACCESS, bool RESIDUAL, int UNROLL>
__global__ void __launch_bounds__(THREADS) dropout_kernel(const __grid_constant__ DropoutArgs a, const __grid_constant__ Numbers numbers, long long elements)
{
    chained();
    const T* x = static_cast<const T*>(a.x.data);
    const T* residual = static_cast<const T*>(a.residual.data);
    T* y = static_cast<T*>(a.y.data);
    const unsigned long long offset = a.offset + (a.step != nullptr ? static_cast<unsigned long long>(*a.step) : 0ull);
    const long long first = static_cast<long long>(blockIdx.x) * (THREADS * UNROLL) + threadIdx.x;
    if constexpr (ACCESS != SINGLE) {
        // blocks whose groups are all whole: every load is under way before the first is used
        if ((static_cast<long long>(blockIdx.x) + 1) * (THREADS * UNROLL * GROUP) <= elements) {
            Eight<T> vx[UNROLL], vr[UNROLL];
            T* to[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const long long i = (first + u * THREADS) * GROUP;
                long long at = i, atResidual = i, atY = i;
                if constexpr (ACCESS == ROWS) {
                    const long long row = (elements >> 32) == 0 ? static_cast<unsigned>(i) / static_cast<unsigned>(a.channels) : i / a.channels;
                    const int column = static_cast<int>(i - row * a.channels);
                    at = row * a.x.stride + column;
                    atResidual = row * a.residual.stride + column;
                    atY = row * a.y.stride + column;
                }
                vx[u] = loadEight<T>(x + at);
                if constexpr (RESIDUAL) vr[u] = loadEight<T>(residual + atResidual);
                to[u] = y + atY;
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                uint32_t word[4];
                philox(first + u * THREADS, offset, numbers, word);
                float f[GROUP], r[GROUP];
                unpackEight<T>(vx[u], f);
                if constexpr (RESIDUAL) unpackEight<T>(vr[u], r);
#pragma unroll
                for (int j = 0; j < GROUP; ++j) {
                    // (selected, not multiplied: a dropped infinity or NaN is a zero)
                    f[j] = kept(word, j, numbers.cut) ? f[j] * numbers.scale : 0.f;
                    if constexpr (RESIDUAL) f[j] += r[j];
                }
#pragma unroll
                for (int k = 0; k < GROUP / WIDE<T>; ++k)
                    store<T, WIDE<T>>(to[u] + k * WIDE<T>, pack<T, WIDE<T>>(*reinterpret_cast<const float (*)[WIDE<T>]>(&f[k * WIDE<T>])));
            }
            return;
        }
    }
    for (int u = 0; u < UNROLL; ++u) {
        const long long group = first + u * THREADS, i = group * GROUP;
        if (i >= elements) break;
        uint32_t word[4];
        philox(group, offset, numbers, word);
        long long row = i / a.channels;
        int column = static_cast<int>(i - row * a.channels);
#pragma unroll
        for (int j = 0; j < GROUP; ++j) {
            if (i + j >= elements) break;
            float f = kept(word, j, numbers.cut) ? Element<T>::to(x[row * a.x.stride + column]) * numbers.scale : 0.f;
            if constexpr (RESIDUAL) f += Element<T>::to(residual[row * a.residual.stride + column]);
            y[row * a.y.stride + column] = Element<T>::from(f);
            if (++column == a.channels) {
                column = 0;
                ++row;
            }
        }
    }
}

template <class T>
cudaError_t dropout(const DropoutArgs& a, cudaStream_t stream)
{
    const long long elements = a.rows * a.channels, groups = (elements + GROUP - 1) / GROUP;
    auto aligned = [&](const Rows& r) { return r.data == nullptr || (reinterpret_cast<uintptr_t>(r.data) & 15) == 0; };
    auto dense = [&](const Rows& r) { return r.data == nullptr || r.stride == a.channels; };
    auto apart = [&](const Rows& r) { return r.data == nullptr || r.stride % WIDE<T> == 0; };
    const bool all = aligned(a.x) && aligned(a.residual) && aligned(a.y);
    const int access = all && dense(a.x) && dense(a.residual) && dense(a.y)                                          ? FLAT
                       : all && a.channels % GROUP == 0 && apart(a.x) && apart(a.residual) && apart(a.y) ? ROWS
                                                                                                                    : SINGLE;
    Numbers numbers;
    for (uint32_t round = 0; round < 10; ++round) {
        numbers.low[round] = static_cast<uint32_t>(a.seed) + round * 0x9E3779B9u;
        numbers.high[round] = static_cast<uint32_t>(a.seed >> 32) + round * 0xBB67AE85u;
    }
    numbers.cut = a.cut << 16;
    numbers.scale = static_cast<float>(65536.0 / (65536u - a.cut));
    auto go = [&](auto* kernel, int unroll) {
        const long long blocks = (groups + THREADS * unroll - 1) / (THREADS * unroll);
        if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
        launchChained(kernel, static_cast<unsigned>(blocks), THREADS, 0, stream, 1, a, numbers, elements);
        return cudaGetLastError();
    };
    constexpr int UNROLL = sizeof(T) == 2 ? 4 : 2;
    auto pick = [&](auto residual) {
        constexpr bool R = decltype(residual)::value;
        constexpr int U = R ? UNROLL / 2 : UNROLL;
        return access == FLAT ? go(dropout_kernel<T, FLAT, R, U>, U) : access == ROWS ? go(dropout_kernel<T, ROWS, R, U>, U) : go(dropout_kernel<T, SINGLE, R, 1>, 1);
    };
    return a.residual.data != nullptr ? pick(std::true_type()) : pick(std::false_type());
}

} // namespace

cudaError_t launchDropout(const DropoutArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    if (a.cut >= 65536) {   // nothing is kept: zeros, or the residual as if it were the input and all of it were kept
        const size_t bytes = typeBytes(a.type);
        if (a.residual.data == nullptr) return cudaMemset2DAsync(a.y.data, a.y.stride * bytes, 0, a.channels * bytes, a.rows, stream);
        DropoutArgs all = a;
        all.x = a.residual;
        all.residual = {};
        all.cut = 0;
        return launchDropout(all, stream);
    }
    return a.type == TYPE_FLOAT ? dropout<float>(a, stream) : a.type == TYPE_HALF ? dropout<__half>(a, stream) : dropout<__nv_bfloat16>(a, stream);
}

} // namespace kernel
} // namespace qmlp
