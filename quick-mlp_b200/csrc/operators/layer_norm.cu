// Layer norm over the rows of a feature matrix, and its gradients.
//
//   mean = sum x / C     deviation^2 = sum (x - mean)^2 / C + epsilon     u = (x - mean) / deviation     y = u w + b
//   dx = (g - mean(g) - u mean(g u)) / deviation   with g = dy w        dw = sum over rows of dy u        db = sum over rows of dy
//
// A row is held in the registers of G threads (8 or 32 lanes of a warp, or a block of 64 to 1024), EPT elements each, so that it
// is read once: the variance is summed from the centred values, not from a difference of squares. All sums are fp32.
// Rows of a block of their own (more than 512 channels) come through a ring of bulk copies in shared memory. What bounds the kernels is DRAM;
// on the way there it was instructions (two fp32 operations per instruction, pairs converted at once), L1 (parameters in
// registers) and the latency of a row's sums (one exchange through shared memory per row, the row's statistics fetched ahead).
// 32768 x 4096 bfloat16: forward 87 us, 6.2 TB/s; adjoint 134 us + 4 us for the parameters' sums, 5.8 TB/s.
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

// The elements of a thread: EPT of a row, VEC side by side; number k (in pairs: k, k + 1) is element (k / VEC * G + lane) * VEC + k % VEC.
template <class T, int VEC, int G, int EPT>
__device__ __forceinline__ void fetchRow(const T* row, int lane, int channels, bool active, float2 (&v)[EPT / 2])
{
    Pack<T, VEC> p[EPT / VEC];
#pragma unroll
    for (int n = 0; n < EPT / VEC; ++n) {
        const int c = (n * G + lane) * VEC;
        p[n] = {};
        if (active && c < channels) p[n] = load<T, VEC>(row + c);
    }
#pragma unroll
    for (int n = 0; n < EPT / VEC; ++n) unpack<T, VEC>(p[n], reinterpret_cast<float (*)[VEC]>(&v[0])[n]);
}
template <class T, int VEC, int G, int EPT>
__device__ __forceinline__ void storeRow(T* row, int lane, int channels, const float2 (&v)[EPT / 2])
{
#pragma unroll
    for (int n = 0; n < EPT / VEC; ++n) {
        const int c = (n * G + lane) * VEC;
        if (c < channels) store<T, VEC>(row + c, pack<T, VEC>(reinterpret_cast<const float (*)[VEC]>(&v[0])[n]));
    }
}
// zero where an element lies behind the row's last
template <int VEC, int G, int EPT>
__device__ __forceinline__ void clearBehind(int lane, int channels, float2 (&v)[EPT / 2])
{
#pragma unroll
    for (int n = 0; n < EPT / VEC; ++n)
        if ((n * G + lane) * VEC >= channels) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) reinterpret_cast<float*>(&v[0])[n * VEC + i] = 0.f;
        }
}
template <int N>
__device__ __forceinline__ float pairSum(const float2 (&v)[N])
{
    float2 s = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) s = add2(s, v[i]);
    return s.x + s.y;
}

// Mean and variance of a row whose elements `v` are centred on the way. Each warp has its own mean first, so that one exchange through
// shared memory does for both: sum (x - mean)^2 = sum over warps of (squares about the warp's mean + count * (warp's mean - mean)^2).
template <int VEC, int G, int EPT>
struct Moments {
    static constexpr int LANES = G < 32 ? G : 32;
    float invC, invCount;        // elements of the row; of this warp (group of lanes), 0 if it has none
    float otherCount = 0.f, otherInv = 0.f;   // of warp `lane`
    float* shared;               // 2 x 64 floats
    int half = 0;
    __device__ __forceinline__ Moments(int lane, int channels, float* memory) : shared(memory)
    {
        float count = 0.f;
#pragma unroll
        for (int n = 0; n < EPT / VEC; ++n) count += (n * G + lane) * VEC < channels ? static_cast<float>(VEC) : 0.f;
        count = groupSum<LANES>(count);
        invC = 1.f / static_cast<float>(channels);
        invCount = count > 0.f ? 1.f / count : 0.f;
        if constexpr (G > 32) {
            constexpr int WARPS = G / 32;
            const int l = threadIdx.x & 31;
            if (l == 0) shared[threadIdx.x >> 5] = count;
            __syncthreads();
            otherCount = l < WARPS ? shared[l] : 0.f;
            otherInv = otherCount > 0.f ? 1.f / otherCount : 0.f;
            __syncthreads();
        }
    }
    __device__ __forceinline__ void operator()(int lane, int channels, float2 (&v)[EPT / 2], float& mean, float& variance)
    {
        const float sum = groupSum<LANES>(pairSum(v)), own = sum * invCount;
        float2 s = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i) v[i] = add2(v[i], both(-own));
        clearBehind<VEC, G, EPT>(lane, channels, v);
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i) s = fma2(v[i], v[i], s);
        float squares = groupSum<LANES>(s.x + s.y);
        mean = own;
        if constexpr (G > 32) {
            constexpr int WARPS = G / 32;
            float* at = shared + half * 64;
            half ^= 1;
            const int l = threadIdx.x & 31, warp = threadIdx.x >> 5;
            if (l == 0) *reinterpret_cast<float2*>(at + 2 * warp) = make_float2(sum, squares);
            __syncthreads();
            const float2 other = l < WARPS ? *reinterpret_cast<const float2*>(at + 2 * l) : make_float2(0.f, 0.f);
            mean = groupSum<WARPS>(other.x) * invC;
            if constexpr (WARPS < 32) mean = __shfl_sync(0xffffffffu, mean, 0);
            const float d = fmaf(other.x, otherInv, -mean);
            squares = groupSum<WARPS>(fmaf(d * d, otherCount, other.y));
            if constexpr (WARPS < 32) squares = __shfl_sync(0xffffffffu, squares, 0);
#pragma unroll
            for (int i = 0; i < EPT / 2; ++i) v[i] = add2(v[i], both(own - mean));
        }
        variance = squares * invC;
    }
};

// The parameters of a thread's elements: kept in registers where these allow it, or read from L1 when they are used. (Reading both
// vectors for every row of 4096 bfloat16 keeps L1 82 % busy and was slower: 131 us for 32768 rows.)
template <int VEC, int G, int EPT>
struct Parameters {
    static constexpr bool KEEP = G <= 256;
    float kept[KEEP ? EPT : 1];
    Vector source;
    float otherwise;
    int lane, channels;
    bool wide;
    __device__ __forceinline__ Parameters(const Vector& v, float none, int l, int c) : source(v), otherwise(none), lane(l), channels(c)
    {
        wide = VEC % 4 == 0 && v.type == TYPE_FLOAT && (reinterpret_cast<uintptr_t>(v.data) & 15) == 0;
        if constexpr (KEEP) {
#pragma unroll
            for (int n = 0; n < EPT / VEC; ++n) read(n, *reinterpret_cast<float (*)[VEC]>(&kept[n * VEC]));
        }
    }
    __device__ __forceinline__ void read(int n, float (&f)[VEC]) const
    {
        const int c = (n * G + lane) * VEC;
        if (source.data != nullptr && c < channels) {
            if (wide) {   // (channels is a multiple of VEC)
#pragma unroll
                for (int i = 0; i + 3 < VEC; i += 4) *reinterpret_cast<float4*>(&f[i]) = *reinterpret_cast<const float4*>(static_cast<const float*>(source.data) + c + i);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = element(source, c + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = otherwise;
        }
    }
    __device__ __forceinline__ void get(int n, float (&f)[VEC]) const
    {
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] = kept[n * VEC + i];
        } else {
            read(n, f);
        }
    }
    __device__ __forceinline__ void get(float2 (&f)[EPT / 2]) const
    {
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < EPT / 2; ++i) f[i] = make_float2(kept[2 * i], kept[2 * i + 1]);
        } else {
#pragma unroll
            for (int n = 0; n < EPT / VEC; ++n) read(n, reinterpret_cast<float (*)[VEC]>(&f[0])[n]);
        }
    }
};

// Rows on their way to a block of one row: bulk copies ahead of the row that is worked on, into a ring of `stages` slots in
// shared memory. What is in flight then does not depend on what the threads are doing, nor on their registers.
// A thread that gives up a wait waits no more. The one that issues the copies then issues no more either, and before the block ends those that were
// under way land, or are waited for to the limit once more. (Place and phase of that moment lie in shared memory: registers, or a flag that
// is looked at before every copy, cost the adjoint 4 to 9 %.) The rows are wrong then, and the status says so.
constexpr int RING_MAX = 8;
struct Ring {
    uint32_t slots, bars, slotBytes, rowBytes;
    int stages, stage = 0, phase = 0;
    bool ok = true;
    __device__ __forceinline__ Ring() {}
    // `matrices` rows per slot; called by all threads, ends in a barrier
    __device__ __forceinline__ Ring(unsigned char* memory, int count, int matrices, uint32_t bytes)
        : slots(smemAddress(memory) + 128), bars(smemAddress(memory)), slotBytes(matrices * bytes), rowBytes(bytes), stages(count)
    {
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) barrierInit(bars + i * 8, 1);
            barrierInitDone();
        }
        __syncthreads();
    }
    __device__ __forceinline__ void issue(int at, const void* first, const void* second) const
    {
        barrierExpect(bars + at * 8, slotBytes);
        bulkLoad(slots + at * slotBytes, first, rowBytes, bars + at * 8);
        if (second != nullptr) bulkLoad(slots + at * slotBytes + rowBytes, second, rowBytes, bars + at * 8);
    }
    // offset of the slot whose row is there now
    __device__ __forceinline__ uint32_t await(unsigned char* memory)
    {
        if (ok && !barrierWait(bars + stage * 8, phase)) {
            ok = false;
            if (threadIdx.x == 0) *reinterpret_cast<int*>(memory + RING_MAX * 8) = stage * 2 + phase;
        }
        return 128 + stage * slotBytes;
    }
    // after a wait was given up
    __device__ __forceinline__ void land(unsigned char* memory, int* status) const
    {
        atomicOr(status, 1);
        if (threadIdx.x != 0) return;
        const int at = *reinterpret_cast<const int*>(memory + RING_MAX * 8);
        for (int i = 0; i < stages; ++i) barrierWait(bars + i * 8, (i < (at >> 1) ? 1 : 0) ^ (at & 1));
    }
    __device__ __forceinline__ void advance()
    {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1;
        }
    }
};

// blocks per SM that the registers have to allow
__host__ __device__ constexpr int perSM(int g) { return g <= 32 ? 2 : g <= 256 ? 512 / g : 1; }
__host__ __device__ constexpr int forwardPerSM(int g) { return g <= 32 ? 3 : g <= 256 ? 768 / g : 1024 / g; }

template <class T, int VEC, int G, int EPT, bool RINGED>
__global__ void __launch_bounds__(threadsFor(G), forwardPerSM(G)) layer_norm_forward_kernel(const __grid_constant__ LayerNormArgs a)
{
    chained();
    constexpr int GROUPS = threadsFor(G) / G;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ __align__(8) float shared[2 * 64];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const T* x = static_cast<const T*>(a.x.data);
    T* y = static_cast<T*>(a.y.data);
    const long long step = static_cast<long long>(gridDim.x) * GROUPS;
    long long row = static_cast<long long>(blockIdx.x) * GROUPS + group;
    Ring ring = [&] {
        if constexpr (RINGED) return Ring(dynamic, a.ringStages, 1, a.channels * sizeof(T));
        else return Ring();
    }();
    if (RINGED && threadIdx.x == 0)
        for (int i = 0; i < a.ringStages && row + i * step < a.rows; ++i) ring.issue(i, x + (row + i * step) * a.x.stride, nullptr);
    const Parameters<VEC, G, EPT> w(a.weight, 1.f, lane, a.channels), b(a.bias, 0.f, lane, a.channels);
    Moments<VEC, G, EPT> moments(lane, a.channels, shared);
    for (; row - group < a.rows; row += step) {
        const bool active = row < a.rows;
        float2 v[EPT / 2], f[EPT / 2];
        fetchRow<T, VEC, G, EPT>(RINGED ? reinterpret_cast<const T*>(dynamic + ring.await(dynamic)) : x + row * a.x.stride, lane, a.channels, active, v);
        float mean, variance;
        moments(lane, a.channels, v, mean, variance);
        if constexpr (RINGED) {   // (behind the barrier of the sums: the slot has been read)
            if (threadIdx.x == 0 && ring.ok && row + a.ringStages * step < a.rows) ring.issue(ring.stage, x + (row + a.ringStages * step) * a.x.stride, nullptr);
            ring.advance();
        }
        const float rstd = rsqrtf(variance + a.epsilon);
        if (!active) continue;   // (whole rows: the lanes of a row leave together, the row's sums are complete)
        if (a.stats != nullptr && lane == 0) {
            a.stats[row] = mean;
            a.stats[a.rows + row] = rstd;
        }
        w.get(f);
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i) v[i] = mul2(mul2(v[i], both(rstd)), f[i]);
        b.get(f);
#pragma unroll
        for (int i = 0; i < EPT / 2; ++i) v[i] = add2(v[i], f[i]);
        storeRow<T, VEC, G, EPT>(y + row * a.y.stride, lane, a.channels, v);
    }
    if (RINGED && !ring.ok) ring.land(dynamic, a.status);
}

// VEC elements of a row in the adjoint, from the packed x and dy: u = (x - mean) / deviation, d = dy, g = dy w
template <class T, int VEC>
struct Piece {
    static constexpr int N = (VEC + 1) / 2;
    float2 u[N], d[N], g[N];
    __device__ __forceinline__ Piece(const Pack<T, VEC>& x, const Pack<T, VEC>& dy, const float* w, float mean, float rstd)
    {
        float fx[2 * N] = {}, fd[2 * N] = {};
        unpack<T, VEC>(x, *reinterpret_cast<float (*)[VEC]>(fx));
        unpack<T, VEC>(dy, *reinterpret_cast<float (*)[VEC]>(fd));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u[i] = mul2(add2(make_float2(fx[2 * i], fx[2 * i + 1]), both(-mean)), both(rstd));   // (elements behind the row: whatever, their dy is zero)
            d[i] = make_float2(fd[2 * i], fd[2 * i + 1]);
            g[i] = mul2(d[i], make_float2(w[2 * i], VEC > 1 ? w[2 * i + 1] : 0.f));
        }
    }
};

// Between its sums and its result a row is held packed, and u and g are formed a second time: unpacked they would take twice the registers.
// Blocks of 1024 threads have 64 registers each: they read the row a second time instead.
// 32768 x 4096 bfloat16: 134 us, 6.0 TB/s (blocks that take two rows per step and share the barrier were slower: 159 us against 143 then).
template <class T, int VEC, int G, int EPT, bool RINGED>
__global__ void __launch_bounds__(threadsFor(G), perSM(G)) layer_norm_adjoint_kernel(const __grid_constant__ LayerNormArgs a)
{
    chained();
    constexpr int THREADS = threadsFor(G), GROUPS = THREADS / G, NV = EPT / VEC;
    constexpr bool TWICE = G == 1024;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ float shared[2 * 32 * 2];
    int half = 0;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float invC = 1.f / static_cast<float>(a.channels);
    const T *x = static_cast<const T*>(a.x.data), *dy = static_cast<const T*>(a.gradY.data);
    T* dx = static_cast<T*>(a.gradX.data);
    const long long step = static_cast<long long>(gridDim.x) * GROUPS;
    long long row = static_cast<long long>(blockIdx.x) * GROUPS + group;
    Ring ring = [&] {
        if constexpr (RINGED) return Ring(dynamic, a.ringStages, 2, a.channels * sizeof(T));
        else return Ring();
    }();
    if (RINGED && threadIdx.x == 0)
        for (int i = 0; i < a.ringStages && row + i * step < a.rows; ++i) ring.issue(i, x + (row + i * step) * a.x.stride, dy + (row + i * step) * a.gradY.stride);
    const Parameters<VEC, G, EPT> w(a.weight, 1.f, lane, a.channels);
    float2 dw[EPT / 2] = {}, db[EPT / 2] = {};
    float nextMean, nextRstd;   // on their way for the row after: their latency would be every row's
    auto fetchStats = [&](long long r) {
        nextMean = r < a.rows ? a.stats[r] : 0.f;
        nextRstd = r < a.rows ? a.stats[a.rows + r] : 0.f;
    };
    fetchStats(row);
    for (; row - group < a.rows; row += step) {
        const bool active = row < a.rows;   // (rows behind the last: zeros, which add nothing)
        const float mean = nextMean, rstd = nextRstd;
        fetchStats(row + step);
        const T *rowX = x + row * a.x.stride, *rowY = dy + row * a.gradY.stride;
        if constexpr (RINGED) {
            const unsigned char* slot = dynamic + ring.await(dynamic);
            rowX = reinterpret_cast<const T*>(slot);
            rowY = reinterpret_cast<const T*>(slot + ring.rowBytes);
        }
        Pack<T, VEC> px[NV], py[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * G + lane) * VEC;
            px[n] = py[n] = {};
            if (active && c < a.channels) {
                px[n] = load<T, VEC>(rowX + c);
                py[n] = load<T, VEC>(rowY + c);
            }
        }
        float2 s0 = {0.f, 0.f}, s1 = {0.f, 0.f};
        if constexpr (VEC > 1) {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                float fw[VEC];
                w.get(n, fw);
                const Piece<T, VEC> p(px[n], py[n], fw, mean, rstd);
#pragma unroll
                for (int i = 0; i < VEC / 2; ++i) {
                    float2 &sw = dw[n * VEC / 2 + i], &sb = db[n * VEC / 2 + i];
                    sw = fma2(p.d[i], p.u[i], sw);
                    sb = add2(sb, p.d[i]);
                    s0 = add2(s0, p.g[i]);
                    s1 = fma2(p.g[i], p.u[i], s1);
                }
            }
        } else {
            float *sw = reinterpret_cast<float*>(dw), *sb = reinterpret_cast<float*>(db);
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                float fw[1];
                w.get(n, fw);
                const float d = Element<T>::to(py[n].v[0]), u = (Element<T>::to(px[n].v[0]) - mean) * rstd, g = d * fw[0];
                sw[n] = fmaf(d, u, sw[n]);
                sb[n] += d;
                s0.x += g;
                s1.x = fmaf(g, u, s1.x);
            }
        }
        float sums[2] = {s0.x + s0.y, s1.x + s1.y};
        if (dx != nullptr) rowSum<G, 2>(sums, shared, half);
        else if (RINGED) __syncthreads();
        auto release = [&] {   // behind a barrier: the slot has been read
            const long long after = row + a.ringStages * step;
            if (threadIdx.x == 0 && ring.ok && after < a.rows) ring.issue(ring.stage, x + after * a.x.stride, dy + after * a.gradY.stride);
            ring.advance();
        };
        if constexpr (RINGED && !TWICE) release();
        if (dx != nullptr && active) {
            const float m0 = sums[0] * invC, m1 = sums[1] * invC;
            T* out = dx + row * a.gradX.stride;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int c = (n * G + lane) * VEC;
                if (c >= a.channels) continue;
                if constexpr (TWICE) {
                    px[n] = load<T, VEC>(rowX + c);
                    py[n] = load<T, VEC>(rowY + c);
                }
                float f[VEC], fw[VEC];
                w.get(n, fw);
                if constexpr (VEC > 1) {
                    const Piece<T, VEC> p(px[n], py[n], fw, mean, rstd);
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        const float2 v = mul2(add2(fma2(p.u[i], both(-m1), p.g[i]), both(-m0)), both(rstd));
                        f[2 * i] = v.x;
                        f[2 * i + 1] = v.y;
                    }
                } else {
                    const float u = (Element<T>::to(px[n].v[0]) - mean) * rstd;
                    f[0] = (fmaf(-u, m1, Element<T>::to(py[n].v[0]) * fw[0]) - m0) * rstd;
                }
                store<T, VEC>(out + c, pack<T, VEC>(f));
            }
        }
        if constexpr (RINGED && TWICE) {
            __syncthreads();
            release();
        }
    }
    if (RINGED && !ring.ok) ring.land(dynamic, a.status);
    if (a.partial == nullptr) return;
    float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.channels;
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const int c = (i / VEC * G + lane) * VEC + i % VEC;
            if (c < a.channels) {
                out[c] = reinterpret_cast<const float*>(dw)[i];
                out[a.channels + c] = reinterpret_cast<const float*>(db)[i];
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
                    sumW[k] = (r == 0 ? 0.f : sumW[k]) + reinterpret_cast<const float*>(dw)[i];
                    sumB[k] = (r == 0 ? 0.f : sumB[k]) + reinterpret_cast<const float*>(db)[i];
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
    chained();
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
    chained();
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
    chained();
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
    chained();
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

// A kernel with a ring of rows: as many slots as `perSM` blocks on an SM have room for, at least one (a slot of two rows of 16384
// floats takes 128 KB).
template <class K>
cudaError_t launchRinged(K kernel, LayerNormArgs a, int matrices, unsigned blocks, int threads, int perSM, cudaStream_t stream)
{
    constexpr int SHARED = 224 * 1024;
    const int slot = matrices * a.channels * typeBytes(a.type);
    a.ringStages = std::max(1, std::min(RING_MAX, (SHARED / perSM - 2048) / slot));
    const int bytes = 128 + a.ringStages * slot;
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), SHARED);
    if (e != cudaSuccess) return e;
    launchChained(kernel, blocks, threads, bytes, stream, 1, a);
    return cudaGetLastError();
}

} // namespace

int layerNormPartials(long long rows, int channels, int, int numSMs) { return static_cast<int>(adjointBlocks(rows, channels, numSMs)); }

cudaError_t launchLayerNormForward(const LayerNormArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        if (a.channels > WIDEST) {
            launchChained(layer_norm_wide_forward_kernel<T>, blocksFor(a.rows, 1, a.numSMs, 2), 1024, 0, stream, 1, a);
            return cudaGetLastError();
        }
        const bool vec = wide(a.x, a.type, a.channels) && wide(a.y, a.type, a.channels);
        return byWidth(a.channels, [&](auto g, auto e) {
            constexpr int G = decltype(g)::value, EPT = decltype(e)::value;
            if constexpr (G > 32) {
                if (vec) return launchRinged(layer_norm_forward_kernel<T, WIDE<T>, G, EPT, true>, a, 1, blocksFor(a.rows, 1, a.numSMs, forwardPerSM(G)), G, forwardPerSM(G), stream);
            }
            const unsigned blocks = blocksFor(a.rows, groupsOf(G), a.numSMs, 2 * forwardPerSM(G));
            if (vec && G <= 32) launchChained(layer_norm_forward_kernel<T, WIDE<T>, G, EPT, false>, blocks, threadsFor(G), 0, stream, 1, a);
            else launchChained(layer_norm_forward_kernel<T, 1, G, EPT, false>, blocks, threadsFor(G), 0, stream, 1, a);
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
                    launchChained(layer_norm_wide_adjoint_kernel<T>, blocksFor(a.rows, 1, a.numSMs, 2), 1024, 0, stream, 1, a);
                    const cudaError_t s = cudaGetLastError();
                    if (s != cudaSuccess) return s;
                }
                if (parameters) launchChained(layer_norm_wide_partial_kernel<T>, dim3((a.channels + 255) / 256, blocks), 256, 0, stream, 1, a);
                return cudaGetLastError();
            }
            const bool vec = wide(a.x, a.type, a.channels) && wide(a.gradY, a.type, a.channels) && wide(a.gradX, a.type, a.channels);
            return byWidth(a.channels, [&](auto g, auto n) {
                constexpr int G = decltype(g)::value, EPT = decltype(n)::value;
                if constexpr (G > 32) {
                    if (vec) return launchRinged(layer_norm_adjoint_kernel<T, WIDE<T>, G, EPT, true>, a, 2, blocks, G, perSM(G), stream);
                }
                if (vec && G <= 32) launchChained(layer_norm_adjoint_kernel<T, WIDE<T>, G, EPT, false>, blocks, threadsFor(G), 0, stream, 1, a);
                else launchChained(layer_norm_adjoint_kernel<T, 1, G, EPT, false>, blocks, threadsFor(G), 0, stream, 1, a);
                return cudaGetLastError();
            });
        });
    }
    if (e != cudaSuccess || !parameters) return e;
    launchChained(layer_norm_parameters_kernel, (2 * a.channels + 31) / 32, dim3(32, 16), 0, stream, 1, a.partial, static_cast<int>(blocks), a.channels, a.gradWeight, a.gradWeightType, a.gradBias, a.gradBiasType);
    return cudaGetLastError();
}

} // namespace kernel
} // namespace qmlp
