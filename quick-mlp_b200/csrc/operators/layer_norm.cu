// Layer norm over the rows of a feature matrix, and its gradients.
//
//   mean = sum x / C     deviation^2 = sum (x - mean)^2 / C + epsilon     u = (x - mean) / deviation     y = u w + b
//   dx = (g - mean(g) - u mean(g u)) / deviation   with g = dy w        dw = sum over rows of dy u        db = sum over rows of dy
//
// A row is held in the registers of G threads (8 or 32 lanes of a warp, or a block of 64 to 1024), EPT elements each, so that it
// is read once: the variance is summed from the centred values, not from a difference of squares. All sums are fp32.
// The gradients of the parameters are sums over rows: a block walks its share of the rows with one fp32 sum per column in
// registers, adds up its row groups in shared memory and leaves one row of partial sums; a second kernel adds those up in a
// fixed order, so the result does not change from run to run. Rows wider than 16384 take three passes over memory instead.
#include "common.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

// sum of one value per thread over the G threads of a row; `lane` is the thread's number in the block. Blocks of one row
// (G > 32) alternate between two halves of `shared` (2 x 32 x N floats), so one barrier per sum is enough.
template <int G, int N>
__device__ __forceinline__ void rowSum(float (&v)[N], float* shared, int& half)
{
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = groupSum<(G < 32 ? G : 32)>(v[n]);
    if constexpr (G > 32) {
        float* s = shared + half * 32 * N;
        half ^= 1;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) s[warp * N + n] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = groupSum<G / 32>(lane < G / 32 ? s[lane * N + n] : 0.f);
        if constexpr (G / 32 < 32) {
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, v[n], 0);
        }
    }
}

__host__ __device__ constexpr int threadsFor(int g) { return g <= 32 ? 256 : g; }

template <class T, int VEC, int G, int EPT>
__global__ void __launch_bounds__(threadsFor(G)) layer_norm_forward_kernel(const __grid_constant__ LayerNormArgs a)
{
    constexpr int NV = EPT / VEC, THREADS = threadsFor(G), GROUPS = THREADS / G;
    __shared__ float shared[2 * 32];
    int half = 0;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float invC = 1.f / static_cast<float>(a.channels);
    // the parameters stay in registers where a block walks many rows
    float w[EPT], b[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int c = (i / VEC * G + lane) * VEC + i % VEC;
        w[i] = a.weight.data != nullptr && c < a.channels ? element(a.weight, c) : 1.f;
        b[i] = a.bias.data != nullptr && c < a.channels ? element(a.bias, c) : 0.f;
    }
    const T* x = static_cast<const T*>(a.x.data);
    T* y = static_cast<T*>(a.y.data);
    for (long long first = static_cast<long long>(blockIdx.x) * GROUPS; first < a.rows; first += static_cast<long long>(gridDim.x) * GROUPS) {
        const long long row = first + group;
        const bool active = row < a.rows;
        float v[EPT];
        float sum[1] = {0.f};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + lane) * VEC;
            float f[VEC] = {};
            if (active && c < a.channels) unpack<T, VEC>(load<T, VEC>(x + row * a.x.stride + c), f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) { v[n * VEC + i] = f[i]; sum[0] += f[i]; }
        }
        rowSum<G, 1>(sum, shared, half);
        const float mean = sum[0] * invC;
        float square[1] = {0.f};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const bool inside = (n * G + lane) * VEC < a.channels;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[n * VEC + i] -= mean;
                square[0] += inside ? v[n * VEC + i] * v[n * VEC + i] : 0.f;
            }
        }
        rowSum<G, 1>(square, shared, half);
        const float rstd = rsqrtf(square[0] * invC + a.epsilon);
        if (!active) continue;   // (whole rows: the lanes of a row leave together, the row's sums are complete)
        if (a.stats != nullptr && lane == 0) {
            a.stats[row] = mean;
            a.stats[a.rows + row] = rstd;
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + lane) * VEC;
            if (c >= a.channels) continue;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = fmaf(v[n * VEC + i] * rstd, w[n * VEC + i], b[n * VEC + i]);
            store<T, VEC>(y + row * a.y.stride + c, pack<T, VEC>(f));
        }
    }
}

template <class T, int VEC, int G, int EPT>
__global__ void __launch_bounds__(threadsFor(G)) layer_norm_adjoint_kernel(const __grid_constant__ LayerNormArgs a)
{
    constexpr int NV = EPT / VEC, THREADS = threadsFor(G), GROUPS = THREADS / G;
    __shared__ float shared[2 * 32 * 2];
    int half = 0;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float invC = 1.f / static_cast<float>(a.channels);
    float w[EPT], dw[EPT], db[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int c = (i / VEC * G + lane) * VEC + i % VEC;
        w[i] = a.weight.data != nullptr && c < a.channels ? element(a.weight, c) : 1.f;
        dw[i] = db[i] = 0.f;
    }
    const T *x = static_cast<const T*>(a.x.data), *dy = static_cast<const T*>(a.gradY.data);
    T* dx = static_cast<T*>(a.gradX.data);
    for (long long first = static_cast<long long>(blockIdx.x) * GROUPS; first < a.rows; first += static_cast<long long>(gridDim.x) * GROUPS) {
        const long long row = first + group;
        const bool active = row < a.rows;
        const float mean = active ? a.stats[row] : 0.f, rstd = active ? a.stats[a.rows + row] : 0.f;
        float u[EPT], g[EPT];
        float sums[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + lane) * VEC;
            const bool inside = active && c < a.channels;
            float f[VEC] = {}, d[VEC] = {};
            if (inside) {
                unpack<T, VEC>(load<T, VEC>(x + row * a.x.stride + c), f);
                unpack<T, VEC>(load<T, VEC>(dy + row * a.gradY.stride + c), d);
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int k = n * VEC + i;
                u[k] = inside ? (f[i] - mean) * rstd : 0.f;
                dw[k] = fmaf(d[i], u[k], dw[k]);
                db[k] += d[i];
                g[k] = d[i] * w[k];
                sums[0] += g[k];
                sums[1] = fmaf(g[k], u[k], sums[1]);
            }
        }
        if (dx == nullptr) continue;
        rowSum<G, 2>(sums, shared, half);
        if (!active) continue;
        const float m0 = sums[0] * invC, m1 = sums[1] * invC;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + lane) * VEC;
            if (c >= a.channels) continue;
            float f[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int k = n * VEC + i;
                f[i] = rstd * (g[k] - m0 - u[k] * m1);
            }
            store<T, VEC>(dx + row * a.gradX.stride + c, pack<T, VEC>(f));
        }
    }
    if (a.partial == nullptr) return;
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const int c = (i / VEC * G + lane) * VEC + i % VEC;
            if (c < a.channels) {
                out[c] = dw[i];
                out[a.channels + c] = db[i];
            }
        }
    } else {
        // the block's row groups, one after the other: every column is added up in the same order each time
        __shared__ float sumW[G * EPT], sumB[G * EPT];
        for (int r = 0; r < GROUPS; ++r) {
            if (group == r) {
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    const int k = i * G + lane;
                    sumW[k] = r == 0 ? dw[i] : sumW[k] + dw[i];
                    sumB[k] = r == 0 ? db[i] : sumB[k] + db[i];
                }
            }
            __syncthreads();
        }
        for (int k = threadIdx.x; k < G * EPT; k += THREADS) {
            const int i = k / G, l = k % G, c = (i / VEC * G + l) * VEC + i % VEC;
            if (c < a.channels) {
                out[c] = sumW[k];
                out[a.channels + c] = sumB[k];
            }
        }
    }
}

// adds up the blocks' partial sums: 32 columns x 16 strided shares of the blocks per thread block
__global__ void __launch_bounds__(512) layer_norm_parameters_kernel(const float* __restrict__ partial, int blocks, int channels, void* gradWeight, int weightType,
                                                                    void* gradBias, int biasType)
{
    __shared__ float shared[16][33];
    const int k = blockIdx.x * 32 + threadIdx.x;   // of 2 x channels
    float sum = 0.f;
    if (k < 2 * channels) {
#pragma unroll 8
        for (int b = threadIdx.y; b < blocks; b += 16) sum += partial[static_cast<long long>(b) * 2 * channels + k];
    }
    shared[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && k < 2 * channels) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += shared[i][threadIdx.x];
        if (k < channels && gradWeight != nullptr) storeElement(gradWeight, weightType, k, sum);
        if (k >= channels && gradBias != nullptr) storeElement(gradBias, biasType, k - channels, sum);
    }
}

// ---- rows wider than the registers of a block ------------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void blockSum(float (&v)[N], float* shared, int& half)
{
    rowSum<1024, N>(v, shared, half);
}
template <class T>
__global__ void __launch_bounds__(1024) layer_norm_wide_forward_kernel(const __grid_constant__ LayerNormArgs a)
{
    __shared__ float shared[2 * 32];
    int half = 0;
    const float invC = 1.f / static_cast<float>(a.channels);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x.data) + row * a.x.stride;
        T* y = static_cast<T*>(a.y.data) + row * a.y.stride;
        float sum[1] = {0.f}, square[1] = {0.f};
        for (int c = threadIdx.x; c < a.channels; c += 1024) sum[0] += Element<T>::to(x[c]);
        blockSum<1>(sum, shared, half);
        const float mean = sum[0] * invC;
        for (int c = threadIdx.x; c < a.channels; c += 1024) {
            const float d = Element<T>::to(x[c]) - mean;
            square[0] = fmaf(d, d, square[0]);
        }
        blockSum<1>(square, shared, half);
        const float rstd = rsqrtf(square[0] * invC + a.epsilon);
        if (a.stats != nullptr && threadIdx.x == 0) {
            a.stats[row] = mean;
            a.stats[a.rows + row] = rstd;
        }
        for (int c = threadIdx.x; c < a.channels; c += 1024) {
            const float w = a.weight.data != nullptr ? element(a.weight, c) : 1.f, b = a.bias.data != nullptr ? element(a.bias, c) : 0.f;
            y[c] = Element<T>::from(fmaf((Element<T>::to(x[c]) - mean) * rstd, w, b));
        }
    }
}
template <class T>
__global__ void __launch_bounds__(1024) layer_norm_wide_adjoint_kernel(const __grid_constant__ LayerNormArgs a)
{
    __shared__ float shared[2 * 32 * 2];
    int half = 0;
    const float invC = 1.f / static_cast<float>(a.channels);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T*>(a.x.data) + row * a.x.stride, *dy = static_cast<const T*>(a.gradY.data) + row * a.gradY.stride;
        T* dx = static_cast<T*>(a.gradX.data) + row * a.gradX.stride;
        const float mean = a.stats[row], rstd = a.stats[a.rows + row];
        float sums[2] = {0.f, 0.f};
        for (int c = threadIdx.x; c < a.channels; c += 1024) {
            const float g = Element<T>::to(dy[c]) * (a.weight.data != nullptr ? element(a.weight, c) : 1.f);
            sums[0] += g;
            sums[1] = fmaf(g, (Element<T>::to(x[c]) - mean) * rstd, sums[1]);
        }
        blockSum<2>(sums, shared, half);
        const float m0 = sums[0] * invC, m1 = sums[1] * invC;
        for (int c = threadIdx.x; c < a.channels; c += 1024) {
            const float g = Element<T>::to(dy[c]) * (a.weight.data != nullptr ? element(a.weight, c) : 1.f);
            dx[c] = Element<T>::from(rstd * (g - m0 - (Element<T>::to(x[c]) - mean) * rstd * m1));
        }
    }
}
// column sums of a share of the rows: blockIdx.x = 256 columns, blockIdx.y = share
template <class T>
__global__ void __launch_bounds__(256) layer_norm_wide_partial_kernel(const __grid_constant__ LayerNormArgs a)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.channels) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = Element<T>::to(static_cast<const T*>(a.gradY.data)[row * a.gradY.stride + c]);
        const float u = (Element<T>::to(static_cast<const T*>(a.x.data)[row * a.x.stride + c]) - a.stats[row]) * a.stats[a.rows + row];
        dw = fmaf(d, u, dw);
        db += d;
    }
    float* out = a.partial + static_cast<long long>(blockIdx.y) * 2 * a.channels;
    out[c] = dw;
    out[a.channels + c] = db;
}

// ---- launch ------------------------------------------------------------------------------------------------------------------
constexpr int WIDEST = 16384;   // 1024 threads x 16 elements

unsigned blocksFor(long long rows, int groups, int numSMs, int perSM)
{
    const long long wanted = (rows + groups - 1) / groups, most = static_cast<long long>(numSMs) * perSM;
    return static_cast<unsigned>(std::max<long long>(1, std::min(wanted, most)));
}
// blocks per SM of a kernel of one row per G threads: what the registers allow
constexpr int perSM(int g) { return g <= 32 ? 2 : g <= 256 ? 512 / g : 1; }
constexpr int groupsOf(int g) { return g <= 32 ? 256 / g : 1; }

// calls f<G, EPT>() for a row of `channels` elements
template <class F>
cudaError_t byWidth(int channels, F&& f)
{
    if (channels <= 64) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
    if (channels <= 256) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
    if (channels <= 512) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 16>());
    if (channels <= 1024) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
    if (channels <= 2048) return f(std::integral_constant<int, 128>(), std::integral_constant<int, 16>());
    if (channels <= 4096) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 16>());
    if (channels <= 8192) return f(std::integral_constant<int, 512>(), std::integral_constant<int, 16>());
    return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 16>());
}
template <class F>
cudaError_t byType(int type, F&& f)
{
    switch (type) {
    case TYPE_FLOAT: return f(float());
    case TYPE_HALF: return f(__half());
    default: return f(__nv_bfloat16());
    }
}
unsigned adjointBlocks(long long rows, int channels, int numSMs)
{
    if (channels > WIDEST) return static_cast<unsigned>(std::max<long long>(1, std::min<long long>(rows, 64)));
    unsigned blocks = 1;
    byWidth(channels, [&](auto g, auto) {
        blocks = blocksFor(rows, groupsOf(g()), numSMs, perSM(g()));
        return cudaSuccess;
    });
    return blocks;
}

} // namespace

int layerNormPartials(long long rows, int channels, int, int numSMs) { return static_cast<int>(adjointBlocks(rows, channels, numSMs)); }

cudaError_t launchLayerNormForward(const LayerNormArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        if (a.channels > WIDEST) {
            layer_norm_wide_forward_kernel<T><<<blocksFor(a.rows, 1, a.numSMs, 2), 1024, 0, stream>>>(a);
            return cudaGetLastError();
        }
        const bool vec = wide(a.x, a.type, a.channels) && wide(a.y, a.type, a.channels);
        return byWidth(a.channels, [&](auto g, auto e) {
            constexpr int G = decltype(g)::value, EPT = decltype(e)::value;
            const unsigned blocks = blocksFor(a.rows, groupsOf(G), a.numSMs, 2048 / threadsFor(G));
            if (vec) layer_norm_forward_kernel<T, WIDE<T>, G, EPT><<<blocks, threadsFor(G), 0, stream>>>(a);
            else layer_norm_forward_kernel<T, 1, G, EPT><<<blocks, threadsFor(G), 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

cudaError_t launchLayerNormAdjoint(const LayerNormArgs& a, cudaStream_t stream)
{
    const bool parameters = a.gradWeight != nullptr || a.gradBias != nullptr;
    unsigned blocks = 0;   // (no rows: the sums below are over nothing)
    cudaError_t e = cudaSuccess;
    if (a.rows > 0) {
        blocks = adjointBlocks(a.rows, a.channels, a.numSMs);
        e = byType(a.type, [&](auto t) {
            using T = decltype(t);
            if (a.channels > WIDEST) {
                if (a.gradX.data != nullptr) {
                    layer_norm_wide_adjoint_kernel<T><<<blocksFor(a.rows, 1, a.numSMs, 2), 1024, 0, stream>>>(a);
                    const cudaError_t s = cudaGetLastError();
                    if (s != cudaSuccess) return s;
                }
                if (parameters) layer_norm_wide_partial_kernel<T><<<dim3((a.channels + 255) / 256, blocks), 256, 0, stream>>>(a);
                return cudaGetLastError();
            }
            const bool vec = wide(a.x, a.type, a.channels) && wide(a.gradY, a.type, a.channels) && wide(a.gradX, a.type, a.channels);
            return byWidth(a.channels, [&](auto g, auto n) {
                constexpr int G = decltype(g)::value, EPT = decltype(n)::value;
                if (vec) layer_norm_adjoint_kernel<T, WIDE<T>, G, EPT><<<blocks, threadsFor(G), 0, stream>>>(a);
                else layer_norm_adjoint_kernel<T, 1, G, EPT><<<blocks, threadsFor(G), 0, stream>>>(a);
                return cudaGetLastError();
            });
        });
    }
    if (e != cudaSuccess || !parameters) return e;
    layer_norm_parameters_kernel<<<(2 * a.channels + 31) / 32, dim3(32, 16), 0, stream>>>(a.partial, static_cast<int>(blocks), a.channels, a.gradWeight,
                                                                                         a.gradWeightType, a.gradBias, a.gradBiasType);
    return cudaGetLastError();
}

} // namespace kernel
} // namespace qmlp
