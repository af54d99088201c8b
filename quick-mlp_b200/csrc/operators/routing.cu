// Routing rows to experts: the choice of the k best experts of a row, their weights, the order of the chosen slots by expert, and
// the movement of feature rows into that order and back.
//
//   chosen: the k largest logits of a row, ties to the lowest index; NaN counts as the largest, -inf is never chosen
//   weight: softmax over all experts of the row, or over the chosen ones alone; 0 in a slot without an expert
//   slot s = row * k + j; slots sorted by expert (stable) -> order[r] = s, position[s] = r, offsets[e] = first r of expert e
//   adjoint over the chosen: dz_j = w_j (g_j - sum_i g_i w_i);  over all: dz_i = p_i (g of the slot that chose i, or 0, - sum_j g_j w_j)
//
// A row belongs to LANES lanes of 8 logits each (one for 8 experts, a warp for 256; 32 logits each above that). Every round takes
// the maximum over the lanes of one 64-bit key, the order-preserving form of the logit above the complement of its index, so the
// tie goes to the lowest index without a second reduction.
#include "partition.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

// order-preserving: larger floats give larger integers, NaN the largest of all, -inf 0 (never chosen)
__device__ __forceinline__ unsigned orderedKey(float f)
{
    if (f != f) return 0xffffffffu;
    const unsigned u = __float_as_uint(f + 0.f);   // (-0 becomes +0: the two are equal)
    const unsigned key = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return key == 0x007fffffu ? 0u : key;
}
__device__ __forceinline__ float orderedValue(unsigned key)
{
    if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    if (key == 0u) return __uint_as_float(0xff800000u);
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
template <int LANES>
__device__ __forceinline__ unsigned long long groupMax(unsigned long long v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) {
        const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

// the PER logits of lane `lane` of a row, -inf behind the last expert
template <class T, int PER, bool VECTOR>
__device__ __forceinline__ void loadLogits(const T* row, int lane, int experts, float (&z)[PER])
{
    constexpr int W = VECTOR ? WIDE<T> : 1;
#pragma unroll
    for (int i = 0; i < PER; i += W) {
        const int c = lane * PER + i;
        float f[W];
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = __uint_as_float(0xff800000u);
        if (c < experts) unpack<T, W>(load<T, W>(row + c), f);
#pragma unroll
        for (int k = 0; k < W; ++k) z[i + k] = f[k];
    }
}

constexpr int TILE_ITEMS = 4, TILE_SLOTS = TILE_ITEMS * PARTITION_THREADS;   // slots per block, at most

// Ranks the slots of a tile and writes order and position. `expertOf(i)`: expert of the tile's i-th slot, -1: none.
// `start`: where the tile's slots of an expert begin (shared memory), `last`: experts.
template <class F>
__device__ __forceinline__ void placeSlots(const RouteArgs& a, F&& expertOf, long long firstSlot, int slots, const int* start, uint16_t* counts)
{
    int digit[TILE_ITEMS], rank[TILE_ITEMS];
    tileRanks<TILE_ITEMS, PARTITION_WARPS>([&](int i) { return i < slots ? expertOf(i) : -1; }, a.experts, counts, digit, rank);
    for (int d = threadIdx.x; d < a.experts; d += PARTITION_THREADS) warpOffsets<PARTITION_WARPS>(counts, a.experts, d);
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int i = (warp * TILE_ITEMS + k) * 32 + lane;
        if (i >= slots) continue;
        const long long slot = firstSlot + i;
        int to = -1;
        if (digit[k] >= 0) {
            to = start[digit[k]] + counts[warp * a.experts + digit[k]] + rank[k];
            a.order[to] = static_cast<int>(slot);
        }
        a.position[slot] = to;
    }
}

struct RoutePlan {
    int tokensPerTile, tiles;
    size_t counts, before, bytes;
    RoutePlan(long long tokens, int experts, int chosen)
    {
        tokensPerTile = std::max(1, TILE_SLOTS / chosen);
        tiles = static_cast<int>((tokens + tokensPerTile - 1) / tokensPerTile);
        counts = (static_cast<size_t>(experts) * 4 + 255) / 256 * 256;
        before = counts + (static_cast<size_t>(experts) * tiles * 4 + 255) / 256 * 256;
        bytes = before + static_cast<size_t>(experts) * tiles * 4;
    }
};

// One tile of rows per block: choose, weigh, count the chosen experts. With ALONE there is one tile, and the block places its
// slots itself.
template <class T, int LANES, int PER, bool VECTOR, bool ALONE>
__global__ void __launch_bounds__(256) route_choose_kernel(const __grid_constant__ RouteArgs a, int tokensPerTile, int* __restrict__ tileCounts, int tiles)
{
    extern __shared__ int dynamic[];
    float* shWeight = reinterpret_cast<float*>(dynamic);        // TILE_SLOTS
    int* shExpert = dynamic + TILE_SLOTS;                       // TILE_SLOTS
    int* shCount = shExpert + TILE_SLOTS;                       // experts
    const int lane = threadIdx.x % LANES;
    const long long first = static_cast<long long>(blockIdx.x) * tokensPerTile;
    const int tokens = static_cast<int>(min(static_cast<long long>(tokensPerTile), a.tokens - first));
    for (int i = threadIdx.x; i < a.experts; i += 256) shCount[i] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < tokens; t0 += 256 / LANES) {
        const int t = t0 + threadIdx.x / LANES;
        const bool active = t < tokens;
        float z[PER];
        loadLogits<T, PER, VECTOR>(static_cast<const T*>(a.logits.data) + (first + (active ? t : 0)) * a.logits.stride, lane, a.experts, z);
        unsigned key[PER];
        unsigned long long best = 0;
        auto localBest = [&]() {
            best = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const unsigned long long k = (static_cast<unsigned long long>(key[i]) << 32) | (~static_cast<unsigned>(lane * PER + i));
                if (key[i] != 0 && k > best) best = k;
            }
        };
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = orderedKey(z[i]);
        localBest();
        float top = 0.f, total = 0.f;
        for (int j = 0; j < a.chosen; ++j) {
            const unsigned long long m = groupMax<LANES>(best);
            const int expert = m == 0 ? -1 : static_cast<int>(~static_cast<unsigned>(m));
            const float value = orderedValue(static_cast<unsigned>(m >> 32));
            if (j == 0) {
                top = m == 0 ? 0.f : value;
                if (!a.normalize) {
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < PER; ++i) s += key[i] != 0 ? expf(z[i] - top) : 0.f;
                    total = groupSum<LANES>(s);
                }
            }
            const float share = m == 0 ? 0.f : expf(value - top);
            if (a.normalize) total += share;
            if (expert >= 0 && expert / PER == lane) {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (expert % PER == i) key[i] = 0;
                localBest();
            }
            if (active && lane == 0) {
                shWeight[t * a.chosen + j] = share;
                shExpert[t * a.chosen + j] = expert;
                if (expert >= 0) atomicAdd(&shCount[expert], 1);
            }
        }
        __syncwarp();
        if (active) {   // the lanes of the row share the division of its slots
            for (int j = lane; j < a.chosen; j += LANES) {
                const int i = t * a.chosen + j;
                const float w = shExpert[i] < 0 ? 0.f : shWeight[i] / total;
                a.weights[first * a.chosen + i] = w;
                a.expert[first * a.chosen + i] = shExpert[i];
            }
        }
    }
    __syncthreads();
    if constexpr (ALONE) {
        __shared__ int warpSums[PARTITION_WARPS];
        uint16_t* counts = reinterpret_cast<uint16_t*>(shCount + a.experts);   // warps x experts
        const int total = blockExclusive(shCount, a.experts, warpSums);
        for (int e = threadIdx.x; e < a.experts; e += 256) a.offsets[e] = shCount[e];
        if (threadIdx.x == 0) a.offsets[a.experts] = total;
        const int slots = tokens * a.chosen;
        for (int i = total + threadIdx.x; i < slots; i += 256) a.order[i] = -1;
        placeSlots(a, [&](int i) { return shExpert[i]; }, 0, slots, shCount, counts);
    } else {
        for (int e = threadIdx.x; e < a.experts; e += 256) tileCounts[static_cast<long long>(e) * tiles + blockIdx.x] = shCount[e];
    }
}

__global__ void __launch_bounds__(PARTITION_THREADS) route_place_kernel(const __grid_constant__ RouteArgs a, int tokensPerTile, const int* __restrict__ tileBefore,
                                                                        const int* __restrict__ totals)
{
    extern __shared__ int dynamic[];
    int* start = dynamic;
    uint16_t* counts = reinterpret_cast<uint16_t*>(dynamic + a.experts);
    __shared__ int warpSums[PARTITION_WARPS];
    for (int e = threadIdx.x; e < a.experts; e += PARTITION_THREADS) start[e] = totals[e];
    __syncthreads();
    const int total = blockExclusive(start, a.experts, warpSums);
    const long long firstSlot = static_cast<long long>(blockIdx.x) * tokensPerTile * a.chosen, all = a.tokens * a.chosen;
    const int slots = static_cast<int>(min(static_cast<long long>(tokensPerTile) * a.chosen, all - firstSlot));
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < a.experts; e += PARTITION_THREADS) a.offsets[e] = start[e];
        if (threadIdx.x == 0) a.offsets[a.experts] = total;
    }
    // the tail of the order, behind the last expert's slots
    for (long long i = total + static_cast<long long>(blockIdx.x) * PARTITION_THREADS + threadIdx.x; i < all; i += static_cast<long long>(gridDim.x) * PARTITION_THREADS)
        a.order[i] = -1;
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += PARTITION_THREADS) start[e] += tileBefore[static_cast<long long>(blockIdx.x) * a.experts + e];
    __syncthreads();
    placeSlots(a, [&](int i) { return a.expert[firstSlot + i]; }, firstSlot, slots, start, counts);
}

template <class T, int LANES, int PER, bool VECTOR>
__global__ void __launch_bounds__(256) route_adjoint_kernel(const __grid_constant__ RouteArgs a)
{
    const int lane = threadIdx.x % LANES;
    const long long t = static_cast<long long>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    const bool active = t < a.tokens;
    const long long row = active ? t : 0;
    float mean = 0.f;
    for (int j = lane; j < a.chosen; j += LANES) {
        const long long i = row * a.chosen + j;
        if (a.expert[i] >= 0) mean = fmaf(a.gradWeights[i], a.weights[i], mean);
    }
    mean = groupSum<LANES>(mean);
    float d[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) d[i] = 0.f;
    if (!a.normalize) {
        float z[PER];
        loadLogits<T, PER, VECTOR>(static_cast<const T*>(a.logits.data) + row * a.logits.stride, lane, a.experts, z);
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) best = max(best, static_cast<unsigned long long>(orderedKey(z[i])));
        const float top = orderedValue(static_cast<unsigned>(groupMax<LANES>(best)));
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            z[i] = z[i] == __uint_as_float(0xff800000u) ? 0.f : expf(z[i] - top);
            s += z[i];
        }
        const float inverse = 1.f / groupSum<LANES>(s);
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] = z[i] == 0.f ? 0.f : -(z[i] * inverse) * mean;
    }
    for (int j = 0; j < a.chosen; ++j) {
        const long long i = row * a.chosen + j;
        const int e = a.expert[i] - lane * PER;
        if (e < 0 || e >= PER) continue;
        const float w = a.weights[i], g = w * (a.gradWeights[i] - mean);
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (e == k) d[k] = g;
    }
    if (!active) return;
    T* out = static_cast<T*>(a.gradLogits.data) + row * a.gradLogits.stride;
    constexpr int W = VECTOR ? WIDE<T> : 1;
#pragma unroll
    for (int i = 0; i < PER; i += W) {
        const int c = lane * PER + i;
        if (c >= a.experts) continue;
        float f[W];
#pragma unroll
        for (int k = 0; k < W; ++k) f[k] = d[i + k];
        store<T, W>(out + c, pack<T, W>(f));
    }
}

// ---- movement of feature rows --------------------------------------------------------------------------------------------
// rows[r] = x[order[r] / chosen], zeros behind the last expert's rows. One access per thread and step.
constexpr int MOVES = 4;
template <class T, int VEC>
__global__ void __launch_bounds__(256) dispatch_kernel(const __grid_constant__ ExchangeArgs a, long long total, int perRow)
{
    const T* x = static_cast<const T*>(a.x.data);
    T* rows = static_cast<T*>(a.rows.data);
    const long long first = blockIdx.x * (256ll * MOVES) + threadIdx.x;
    Pack<T, VEC> v[MOVES];
    long long at[MOVES];
#pragma unroll
    for (int k = 0; k < MOVES; ++k) {
        const long long i = first + k * 256;
        at[k] = -1;
        v[k] = {};
        if (i >= total) continue;
        const long long r = total <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(perRow) : i / perRow;
        const int c = static_cast<int>(i - r * perRow) * VEC, slot = a.order[r];
        at[k] = r * a.rows.stride + c;
        if (slot >= 0 && slot / a.chosen < a.tokens) v[k] = load<T, VEC>(x + static_cast<long long>(slot / a.chosen) * a.x.stride + c);
    }
#pragma unroll
    for (int k = 0; k < MOVES; ++k)
        if (at[k] >= 0) store<T, VEC>(rows + at[k], v[k]);
}

// x[t] = sum over the row's slots of (weight *) rows[position]
template <class T, int VEC, bool WEIGHTED>
__global__ void __launch_bounds__(256) gather_sum_kernel(const __grid_constant__ ExchangeArgs a, Rows rowsIn, Rows out, long long total, int perRow)
{
    const T* rows = static_cast<const T*>(rowsIn.data);
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= total) return;
    const long long t = total <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(perRow) : i / perRow;
    const int c = static_cast<int>(i - t * perRow) * VEC;
    const long long slots = a.tokens * a.chosen;
    float sum[VEC] = {};
    for (int j0 = 0; j0 < a.chosen; j0 += 4) {
        Pack<T, VEC> v[4];
        float w[4];
        bool use[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            use[j] = false;
            if (j0 + j < a.chosen) {
                const long long s = t * a.chosen + j0 + j;
                const int r = a.position[s];
                use[j] = r >= 0 && r < slots;
                w[j] = WEIGHTED ? a.weights[s] : 1.f;
                if (use[j]) v[j] = load<T, VEC>(rows + static_cast<long long>(r) * rowsIn.stride + c);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!use[j]) continue;
            float f[VEC];
            unpack<T, VEC>(v[j], f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) sum[k] = WEIGHTED ? fmaf(w[j], f[k], sum[k]) : sum[k] + f[k];
        }
    }
    store<T, VEC>(static_cast<T*>(out.data) + t * out.stride + c, pack<T, VEC>(sum));
}

// gradients of the combination: G lanes per row read its gradient once per slot (the first time from memory), write the slot's
// row of gradients and add up the slot's product with its row
template <class T, int VEC, int G>
__global__ void __launch_bounds__(256) combine_adjoint_kernel(const __grid_constant__ ExchangeArgs a)
{
    const int lane = threadIdx.x % G;
    const long long t = static_cast<long long>(blockIdx.x) * (256 / G) + threadIdx.x / G, slots = a.tokens * a.chosen;
    const bool active = t < a.tokens;
    const T *rows = static_cast<const T*>(a.rows.data), *dy = static_cast<const T*>(a.gradX.data) + (active ? t : 0) * a.gradX.stride;
    T* out = static_cast<T*>(a.gradRows.data);
    for (int j = 0; j < a.chosen; ++j) {
        const long long s = (active ? t : 0) * a.chosen + j;
        const int r = a.position[s];
        const bool use = active && r >= 0 && r < slots;
        float dot = 0.f;
        if (use) {
            const float w = a.weights[s];
            for (int c = lane * VEC; c < a.channels; c += G * VEC) {
                float g[VEC], f[VEC];
                unpack<T, VEC>(load<T, VEC>(dy + c), g);
                if (a.gradWeights != nullptr) {
                    unpack<T, VEC>(load<T, VEC>(rows + static_cast<long long>(r) * a.rows.stride + c), f);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) dot = fmaf(g[k], f[k], dot);
                }
                if (out != nullptr) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) f[k] = w * g[k];
                    store<T, VEC>(out + static_cast<long long>(r) * a.gradRows.stride + c, pack<T, VEC>(f));
                }
            }
        }
        dot = groupSum<G>(dot);
        if (active && lane == 0 && a.gradWeights != nullptr) a.gradWeights[s] = dot;
    }
}
// zeros behind the last expert's rows: a warp looks at 32 rows and clears those without a slot
template <class T, int VEC>
__global__ void __launch_bounds__(256) clear_tail_kernel(const __grid_constant__ ExchangeArgs a)
{
    T* out = static_cast<T*>(a.gradRows.data);
    const long long slots = a.tokens * a.chosen, first = (static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * 32;
    const int lane = threadIdx.x & 31;
    unsigned empty = __ballot_sync(0xffffffffu, first + lane < slots && a.order[first + lane] < 0);
    for (; empty != 0; empty &= empty - 1) {
        const long long r = first + __ffs(empty) - 1;
        for (int c = lane * VEC; c < a.channels; c += 32 * VEC) store<T, VEC>(out + r * a.gradRows.stride + c, Pack<T, VEC>{});
    }
}

// ---- launch --------------------------------------------------------------------------------------------------------------
template <class F>
cudaError_t byType(int type, F&& f)
{
    switch (type) {
    case TYPE_FLOAT: return f(float());
    case TYPE_HALF: return f(__half());
    default: return f(__nv_bfloat16());
    }
}
// calls f<LANES, PER>() for a number of experts
template <class F>
cudaError_t byExperts(int experts, F&& f)
{
    using I8 = std::integral_constant<int, 8>;
    if (experts <= 8) return f(std::integral_constant<int, 1>(), I8());
    if (experts <= 16) return f(std::integral_constant<int, 2>(), I8());
    if (experts <= 32) return f(std::integral_constant<int, 4>(), I8());
    if (experts <= 64) return f(std::integral_constant<int, 8>(), I8());
    if (experts <= 128) return f(std::integral_constant<int, 16>(), I8());
    if (experts <= 256) return f(std::integral_constant<int, 32>(), I8());
    return f(std::integral_constant<int, 32>(), std::integral_constant<int, 32>());
}

} // namespace

size_t routeBytes(long long tokens, int experts, int chosen)
{
    if (tokens == 0) return 0;
    const RoutePlan p(tokens, experts, chosen);
    return p.tiles == 1 ? 0 : p.bytes;
}

cudaError_t launchRouteForward(const RouteArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaMemsetAsync(a.offsets, 0, (a.experts + 1) * sizeof(int), stream);
    const RoutePlan p(a.tokens, a.experts, a.chosen);
    const bool alone = p.tiles == 1, vec = wide(a.logits, a.type, a.experts);
    int* totals = static_cast<int*>(a.scratch);
    int* counts = reinterpret_cast<int*>(static_cast<unsigned char*>(a.scratch) + p.counts);
    int* before = reinterpret_cast<int*>(static_cast<unsigned char*>(a.scratch) + p.before);
    cudaError_t e = byType(a.type, [&](auto t) {
        using T = decltype(t);
        return byExperts(a.experts, [&](auto l, auto per) {
            constexpr int LANES = decltype(l)::value, PER = decltype(per)::value;
            const size_t bytes = (2 * TILE_SLOTS + a.experts * (alone ? 1 + PARTITION_WARPS : 1)) * sizeof(int);
            auto go = [&](auto kernel) {
                kernel<<<p.tiles, 256, bytes, stream>>>(a, p.tokensPerTile, counts, p.tiles);
                return cudaGetLastError();
            };
            if (vec) return alone ? go(route_choose_kernel<T, LANES, PER, true, true>) : go(route_choose_kernel<T, LANES, PER, true, false>);
            return alone ? go(route_choose_kernel<T, LANES, PER, false, true>) : go(route_choose_kernel<T, LANES, PER, false, false>);
        });
    });
    if (e != cudaSuccess || alone) return e;
    partition_scan_kernel<<<(a.experts + PARTITION_WARPS - 1) / PARTITION_WARPS, PARTITION_THREADS, 0, stream>>>(counts, before, totals, a.experts, p.tiles);
    route_place_kernel<<<p.tiles, PARTITION_THREADS, (1 + PARTITION_WARPS) * a.experts * sizeof(int), stream>>>(a, p.tokensPerTile, before, totals);
    return cudaGetLastError();
}

cudaError_t launchRouteAdjoint(const RouteArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    const bool vec = wide(a.logits, a.type, a.experts) && wide(a.gradLogits, a.type, a.experts);
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        return byExperts(a.experts, [&](auto l, auto per) {
            constexpr int LANES = decltype(l)::value, PER = decltype(per)::value;
            const unsigned blocks = static_cast<unsigned>((a.tokens + 256 / LANES - 1) / (256 / LANES));
            if (vec) route_adjoint_kernel<T, LANES, PER, true><<<blocks, 256, 0, stream>>>(a);
            else route_adjoint_kernel<T, LANES, PER, false><<<blocks, 256, 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

cudaError_t launchDispatch(const ExchangeArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = wide(a.x, a.type, a.channels) && wide(a.rows, a.type, a.channels);
        const int perRow = vec ? a.channels / WIDE<T> : a.channels;
        const long long total = a.tokens * a.chosen * perRow;
        const unsigned blocks = static_cast<unsigned>((total + 256 * MOVES - 1) / (256 * MOVES));
        if (vec) dispatch_kernel<T, WIDE<T>><<<blocks, 256, 0, stream>>>(a, total, perRow);
        else dispatch_kernel<T, 1><<<blocks, 256, 0, stream>>>(a, total, perRow);
        return cudaGetLastError();
    });
}

static cudaError_t launchGatherSum(const ExchangeArgs& a, const Rows& in, const Rows& out, bool weighted, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = wide(in, a.type, a.channels) && wide(out, a.type, a.channels);
        const int perRow = vec ? a.channels / WIDE<T> : a.channels;
        const long long total = a.tokens * perRow;
        const unsigned blocks = static_cast<unsigned>((total + 255) / 256);
        auto go = [&](auto kernel) {
            kernel<<<blocks, 256, 0, stream>>>(a, in, out, total, perRow);
            return cudaGetLastError();
        };
        if (vec) return weighted ? go(gather_sum_kernel<T, WIDE<T>, true>) : go(gather_sum_kernel<T, WIDE<T>, false>);
        return weighted ? go(gather_sum_kernel<T, 1, true>) : go(gather_sum_kernel<T, 1, false>);
    });
}
cudaError_t launchDispatchAdjoint(const ExchangeArgs& a, cudaStream_t stream) { return launchGatherSum(a, a.gradRows, a.gradX, false, stream); }
cudaError_t launchCombine(const ExchangeArgs& a, cudaStream_t stream) { return launchGatherSum(a, a.rows, a.x, true, stream); }

cudaError_t launchCombineAdjoint(const ExchangeArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = wide(a.rows, a.type, a.channels) && wide(a.gradX, a.type, a.channels) && wide(a.gradRows, a.type, a.channels);
        auto go = [&](auto v, auto g) {
            constexpr int VEC = decltype(v)::value, G = decltype(g)::value;
            combine_adjoint_kernel<T, VEC, G><<<static_cast<unsigned>((a.tokens + 256 / G - 1) / (256 / G)), 256, 0, stream>>>(a);
            const cudaError_t e = cudaGetLastError();
            if (e != cudaSuccess || a.gradRows.data == nullptr) return e;
            clear_tail_kernel<T, VEC><<<static_cast<unsigned>((a.tokens * a.chosen + 255) / 256), 256, 0, stream>>>(a);
            return cudaGetLastError();
        };
        if (vec) return a.channels <= 8 * WIDE<T> ? go(std::integral_constant<int, WIDE<T>>(), std::integral_constant<int, 8>())
                                                  : go(std::integral_constant<int, WIDE<T>>(), std::integral_constant<int, 32>());
        return a.channels <= 8 ? go(std::integral_constant<int, 1>(), std::integral_constant<int, 8>()) : go(std::integral_constant<int, 1>(), std::integral_constant<int, 32>());
    });
}

} // namespace kernel
} // namespace qmlp
