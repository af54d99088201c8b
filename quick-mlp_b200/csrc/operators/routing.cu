// Routing rows to experts: the choice of the k best experts of a row, their weights, the order of the chosen slots by expert, and
// the movement of feature rows into that order and back.
//
//   chosen: the k largest logits of a row, ties to the lowest index; NaN counts as the largest, -inf is never chosen
//   weight: softmax over all experts of the row, or over the chosen ones alone; 0 in a slot without an expert
//   slot s = row * k + j; slots sorted by expert (stable) -> order[r] = s, position[s] = r, offsets[e] = first r of expert e
//   adjoint over the chosen: dz_j = w_j (g_j - sum_i g_i w_i);  over all: dz_i = p_i (g of the slot that chose i, or 0, - sum_j g_j w_j)
//
// A row belongs to LANES lanes of 8 logits each (one for 8 experts, a warp for 256; 32 logits each above that). Every round takes
// the maximum over the lanes of one key that holds the logit and its expert.
#include "partition.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

// Keys of logits: larger logits give larger keys, NaN the largest of all, -inf gives 0 (never chosen); below the logit's bits the complement of the
// expert's number, so that the largest key is the first of equal logits. 32 bits hold a 16-bit logit and its expert, floats take 64.
template <class T> struct Key;
template <> struct Key<float> {
    using Type = unsigned long long;
    static __device__ __forceinline__ Type of(float f, int expert)
    {
        const unsigned u = __float_as_uint(f + 0.f);   // (-0 becomes +0: the two are equal)
        const unsigned key = f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
        return key == 0x007fffffu ? 0ull : static_cast<Type>(key) << 32 | ~static_cast<unsigned>(expert);
    }
    static __device__ __forceinline__ float value(Type k)
    {
        const unsigned key = static_cast<unsigned>(k >> 32);
        return __uint_as_float(key == 0xffffffffu ? 0x7fc00000u : (key & 0x80000000u) ? key & 0x7fffffffu : ~key);
    }
    static __device__ __forceinline__ int expert(Type k) { return static_cast<int>(~static_cast<unsigned>(k)); }
};
template <class T, unsigned INF>
struct ShortKey {
    using Type = unsigned;
    static __device__ __forceinline__ Type of(T f, int expert)
    {
        const unsigned u = *reinterpret_cast<const unsigned short*>(&f), magnitude = u & 0x7fffu;
        unsigned key = u > 0x8000u ? ~u & 0xffffu : magnitude | 0x8000u;   // (-0 becomes +0: the two are equal)
        if (magnitude > INF) key = 0xffffu;
        return u == (0x8000u | INF) ? 0u : key << 16 | (0xffffu - expert);
    }
    static __device__ __forceinline__ float value(Type k)
    {
        const unsigned key = k >> 16;
        const unsigned short u = static_cast<unsigned short>(key == 0xffffu ? 0x7fffu : (key & 0x8000u) ? key & 0x7fffu : ~key);
        return Element<T>::to(*reinterpret_cast<const T*>(&u));
    }
    static __device__ __forceinline__ int expert(Type k) { return static_cast<int>(0xffffu - (k & 0xffffu)); }
};
template <> struct Key<__half> : ShortKey<__half, 0x7c00u> {};
template <> struct Key<__nv_bfloat16> : ShortKey<__nv_bfloat16, 0x7f80u> {};

template <int LANES, class K>
__device__ __forceinline__ K groupMax(K v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o /= 2) {
        const K w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

template <class T> __device__ __forceinline__ T minusInfinity() { return Element<T>::from(__uint_as_float(0xff800000u)); }
// the PER logits of lane `lane` of a row, as they lie in memory; -inf behind the last expert
template <class T, int PER, bool VECTOR>
__device__ __forceinline__ void loadLogits(const T* row, int lane, int experts, T (&z)[PER])
{
    constexpr int W = VECTOR ? WIDE<T> : 1;
#pragma unroll
    for (int i = 0; i < PER; i += W) {
        const int c = lane * PER + i;
        Pack<T, W> p;
#pragma unroll
        for (int k = 0; k < W; ++k) p.v[k] = minusInfinity<T>();
        if (c < experts) p = load<T, W>(row + c);
#pragma unroll
        for (int k = 0; k < W; ++k) z[i + k] = p.v[k];
    }
}

// slots per block, at most: a block that is alone takes 1024, else 512, so that the rows of a tile are few passes of a block
constexpr int ALONE_ITEMS = 4, TILE_ITEMS = 2;
constexpr int ALONE_SLOTS = ALONE_ITEMS * PARTITION_THREADS, TILE_SLOTS = TILE_ITEMS * PARTITION_THREADS;
constexpr int TILE_BLOCKS = 148;   // tiles wanted at least: an SM each (a constant, so that the size of the scratch can be asked for without a device)

// Ranks the slots of a tile and writes order and position. `expertOf(i)`: expert of the tile's i-th slot, -1: none.
// `start`: where the tile's slots of an expert begin (shared memory), `last`: experts.
template <int ITEMS, class F>
__device__ __forceinline__ void placeSlots(const RouteArgs& a, F&& expertOf, long long firstSlot, int slots, const int* start, uint16_t* counts)
{
    int digit[ITEMS], rank[ITEMS];
    tileRanks<ITEMS, PARTITION_WARPS>([&](int i) { return i < slots ? expertOf(i) : -1; }, a.experts, counts, digit, rank);
    for (int d = threadIdx.x; d < a.experts; d += PARTITION_THREADS) warpOffsets<PARTITION_WARPS>(counts, a.experts, d);
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (warp * ITEMS + k) * 32 + lane;
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
        // small batches in tiles of 32 rows and more, so that every SM has one: 2048 rows in 4 tiles of 512 took 12.6 us
        const int most = std::max(1, TILE_SLOTS / chosen);
        const long long even = (tokens + TILE_BLOCKS - 1) / TILE_BLOCKS;
        tokensPerTile = tokens * chosen <= ALONE_SLOTS ? ALONE_SLOTS / chosen : static_cast<int>(std::min<long long>(most, (even + 31) / 32 * 32));
        tiles = static_cast<int>((tokens + tokensPerTile - 1) / tokensPerTile);
        counts = (static_cast<size_t>(experts) * 4 + 255) / 256 * 256;
        before = counts + (static_cast<size_t>(experts) * tiles * 4 + 255) / 256 * 256;
        bytes = before + static_cast<size_t>(experts) * tiles * 4;
    }
};

// One tile of rows per block: choose, weigh, count the chosen experts. With ALONE there is one tile, and the block places its
// slots itself. For rows that no thread takes alone: 131072 of 64 half logits, 8 chosen, 38 us. (262147 rows, 2 chosen, in this form 33 us; with 64-bit keys,
// tiles of 1024 slots and no row fetched ahead 60 us.)
template <class T, int LANES, int PER, bool VECTOR, bool ALONE>
__global__ void __launch_bounds__(256) route_choose_kernel(const __grid_constant__ RouteArgs a, int tokensPerTile, int* __restrict__ tileCounts, int tiles)
{
    chained();
    using K = Key<T>;
    constexpr int SLOTS = ALONE ? ALONE_SLOTS : TILE_SLOTS;
    extern __shared__ int dynamic[];
    float* shWeight = reinterpret_cast<float*>(dynamic);        // SLOTS: exp(logit - largest)
    int* shExpert = dynamic + SLOTS;                            // SLOTS
    float* shTotal = reinterpret_cast<float*>(dynamic + 2 * SLOTS);   // SLOTS: of a row
    int* shCount = dynamic + 3 * SLOTS;                         // experts
    const int lane = threadIdx.x % LANES;
    const long long first = static_cast<long long>(blockIdx.x) * tokensPerTile;
    const int tokens = static_cast<int>(min(static_cast<long long>(tokensPerTile), a.tokens - first));
    const T* logits = static_cast<const T*>(a.logits.data) + first * a.logits.stride;
    T next[PER];   // the row after is on its way while one is worked on
    int t = threadIdx.x / LANES;
    loadLogits<T, PER, VECTOR>(logits + (t < tokens ? t : 0) * a.logits.stride, lane, a.experts, next);
    for (int i = threadIdx.x; i < a.experts; i += 256) shCount[i] = 0;
    __syncthreads();
    for (int t0 = 0; t0 < tokens; t0 += 256 / LANES, t += 256 / LANES) {
        const bool active = t < tokens;
        typename K::Type key[PER], best = 0;
        float z[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            key[i] = K::of(next[i], lane * PER + i);
            z[i] = Element<T>::to(next[i]);
            best = key[i] > best ? key[i] : best;
        }
        if (t0 + 256 / LANES < tokens) {
            const int after = t + 256 / LANES;
            loadLogits<T, PER, VECTOR>(logits + (after < tokens ? after : 0) * a.logits.stride, lane, a.experts, next);
        }
        float top = 0.f, total = 0.f;
        for (int j = 0; j < a.chosen; ++j) {
            const typename K::Type m = groupMax<LANES>(best);
            const float value = K::value(m);
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
            best = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (key[i] == m) key[i] = 0;
                best = key[i] > best ? key[i] : best;
            }
            if (active && lane == 0) {
                const int expert = m == 0 ? -1 : K::expert(m);
                shWeight[t * a.chosen + j] = share;
                shExpert[t * a.chosen + j] = expert;
                if (expert >= 0) atomicAdd(&shCount[expert], 1);
            }
        }
        if (active && lane == 0) shTotal[t] = total;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * a.chosen; i += 256) {
        const int expert = shExpert[i];
        a.weights[first * a.chosen + i] = expert < 0 ? 0.f : shWeight[i] / shTotal[i / a.chosen];
        a.expert[first * a.chosen + i] = expert;
    }
    if constexpr (ALONE) {
        __shared__ int warpSums[PARTITION_WARPS];
        uint16_t* counts = reinterpret_cast<uint16_t*>(shCount + a.experts);   // warps x experts
        const int total = blockExclusive(shCount, a.experts, warpSums);
        for (int e = threadIdx.x; e < a.experts; e += 256) a.offsets[e] = shCount[e];
        if (threadIdx.x == 0) a.offsets[a.experts] = total;
        const int slots = tokens * a.chosen;
        for (int i = total + threadIdx.x; i < slots; i += 256) a.order[i] = -1;
        placeSlots<ALONE_ITEMS>(a, [&](int i) { return shExpert[i]; }, 0, slots, shCount, counts);
    } else {
        for (int e = threadIdx.x; e < a.experts; e += 256) tileCounts[static_cast<long long>(e) * tiles + blockIdx.x] = shCount[e];
    }
}

// ---- a row per thread --------------------------------------------------------------------------------------------------------
// Groups of lanes spend most of their instructions on one another (92 per row of 64 experts). Where there are rows enough, a thread keeps a row's
// largest keys in registers, in order, and looks at every logit once; a warp moves its 32 rows through shared memory, 128 bytes of each at a time,
// so that memory is read and written in whole lines (16-byte pieces of a row are exchanged by the row's number against bank conflicts).
// 262147 rows of 64 half logits, 2 chosen: 22 us, adjoint 10 us (groups of 8 lanes: 33 and 19 us).
constexpr int ROWS_CHOSEN = 8, ROWS_EXPERTS = 256;   // most of either
template <class T>
struct RowStage {
    static constexpr int W = WIDE<T>, COLUMNS = 128 / static_cast<int>(sizeof(T));
    unsigned char* mine;   // 32 rows x 128 bytes of this warp
    int lane;
    __device__ __forceinline__ explicit RowStage(unsigned char* memory) : mine(memory + (threadIdx.x >> 5) * 32 * 128), lane(threadIdx.x & 31) {}
    // columns [c0, c0 + COLUMNS) of the rows [0, rows) of `matrix`; -inf behind either
    __device__ __forceinline__ void fetch(const T* matrix, long long stride, long long rows, int c0, int columns)
    {
        const int c = c0 + (lane & 7) * W;
        Pack<T, W> v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
#pragma unroll
            for (int k = 0; k < W; ++k) v[i].v[k] = minusInfinity<T>();
            if (r < rows && c < columns) v[i] = load<T, W>(matrix + r * stride + c);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            store<T, W>(reinterpret_cast<T*>(mine + r * 128 + (((lane & 7) ^ (r & 7)) << 4)), v[i]);
        }
        __syncwarp();
    }
    // piece q of this lane's row
    __device__ __forceinline__ T* piece(int q) const { return reinterpret_cast<T*>(mine + lane * 128 + ((q ^ (lane & 7)) << 4)); }
    __device__ __forceinline__ void put(T* matrix, long long stride, long long rows, int c0, int columns)
    {
        __syncwarp();
        const int c = c0 + (lane & 7) * W;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (r < rows && c < columns) store<T, W>(matrix + r * stride + c, load<T, W>(reinterpret_cast<const T*>(mine + r * 128 + (((lane & 7) ^ (r & 7)) << 4))));
        }
        __syncwarp();
    }
};

template <class T, int CHOSEN>
__global__ void __launch_bounds__(256) route_rows_kernel(const __grid_constant__ RouteArgs a, int tokensPerTile, int* __restrict__ tileCounts, int tiles)
{
    chained();
    using K = Key<T>;
    using Stage = RowStage<T>;
    extern __shared__ __align__(128) unsigned char rowMemory[];   // 8 warps x 32 rows x 128 bytes
    __shared__ int count[ROWS_EXPERTS];
    Stage stage(rowMemory);
    const long long first = static_cast<long long>(blockIdx.x) * tokensPerTile;
    const int tokens = static_cast<int>(min(static_cast<long long>(tokensPerTile), a.tokens - first));
    for (int i = threadIdx.x; i < a.experts; i += 256) count[i] = 0;
    __syncthreads();
    for (int t0 = static_cast<int>(threadIdx.x & ~31u); t0 < tokens; t0 += 256) {   // this warp's 32 rows
        const T* logits = static_cast<const T*>(a.logits.data) + (first + t0) * a.logits.stride;
        typename K::Type best[CHOSEN] = {};
        for (int c0 = 0; c0 < a.experts; c0 += Stage::COLUMNS) {
            stage.fetch(logits, a.logits.stride, tokens - t0, c0, a.experts);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const Pack<T, Stage::W> v = load<T, Stage::W>(stage.piece(q));
#pragma unroll
                for (int i = 0; i < Stage::W; ++i) {
                    typename K::Type key = K::of(v.v[i], c0 + q * Stage::W + i);
#pragma unroll
                    for (int j = 0; j < CHOSEN; ++j) {   // into its place among the largest
                        const typename K::Type high = max(key, best[j]);
                        key = min(key, best[j]);
                        best[j] = high;
                    }
                }
            }
        }
        const float top = best[0] == 0 ? 0.f : K::value(best[0]);
        float total = 0.f, share[CHOSEN];
#pragma unroll
        for (int j = 0; j < CHOSEN; ++j) {
            share[j] = j < a.chosen && best[j] != 0 ? expf(K::value(best[j]) - top) : 0.f;
            total += share[j];
        }
        if (!a.normalize) {
            total = 0.f;
            for (int c0 = 0; c0 < a.experts; c0 += Stage::COLUMNS) {
                if (a.experts > Stage::COLUMNS) stage.fetch(logits, a.logits.stride, tokens - t0, c0, a.experts);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    float f[Stage::W];
                    unpack<T, Stage::W>(load<T, Stage::W>(stage.piece(q)), f);
#pragma unroll
                    for (int i = 0; i < Stage::W; ++i) total += best[0] == 0 || f[i] == __uint_as_float(0xff800000u) ? 0.f : expf(f[i] - top);
                }
            }
        }
        const int t = t0 + (threadIdx.x & 31);
        if (t < tokens) {
#pragma unroll
            for (int j = 0; j < CHOSEN; ++j) {
                if (j >= a.chosen) break;
                const int expert = best[j] == 0 ? -1 : K::expert(best[j]);
                a.weights[(first + t) * a.chosen + j] = expert < 0 ? 0.f : share[j] / total;
                a.expert[(first + t) * a.chosen + j] = expert;
                if (expert >= 0) atomicAdd(&count[expert], 1);
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += 256) tileCounts[static_cast<long long>(e) * tiles + blockIdx.x] = count[e];
}

template <class T, int CHOSEN>
__global__ void __launch_bounds__(256) route_rows_adjoint_kernel(const __grid_constant__ RouteArgs a)
{
    chained();
    using Stage = RowStage<T>;
    extern __shared__ __align__(128) unsigned char rowMemory[];
    Stage stage(rowMemory);
    const long long t0 = static_cast<long long>(blockIdx.x) * 256 + (threadIdx.x & ~31u), t = t0 + (threadIdx.x & 31);
    if (t0 >= a.tokens) return;
    const T* logits = static_cast<const T*>(a.logits.data) + t0 * a.logits.stride;
    T* out = static_cast<T*>(a.gradLogits.data) + t0 * a.gradLogits.stride;
    int expert[CHOSEN];
    float weight[CHOSEN], grad[CHOSEN], mean = 0.f;
#pragma unroll
    for (int j = 0; j < CHOSEN; ++j) {
        const bool have = t < a.tokens && j < a.chosen;
        expert[j] = have ? a.expert[t * a.chosen + j] : -1;
        weight[j] = have ? a.weights[t * a.chosen + j] : 0.f;
        grad[j] = have ? a.gradWeights[t * a.chosen + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < CHOSEN; ++j)
        if (expert[j] >= 0) mean = fmaf(grad[j], weight[j], mean);
    constexpr float NONE = -INFINITY;
    float top = NONE, total = 0.f;
    bool nan = false;
    if (!a.normalize) {
        for (int c0 = 0; c0 < a.experts; c0 += Stage::COLUMNS) {   // largest logit and sum of the exponentials, a piece of the row at a time
            stage.fetch(logits, a.logits.stride, a.tokens - t0, c0, a.experts);
            float high = top;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float f[Stage::W];
                unpack<T, Stage::W>(load<T, Stage::W>(stage.piece(q)), f);
#pragma unroll
                for (int i = 0; i < Stage::W; ++i) {
                    high = fmaxf(high, f[i]);
                    nan = nan || f[i] != f[i];
                }
            }
            if (high == NONE) continue;
            total *= top == NONE ? 0.f : expf(top - high);
            top = high;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float f[Stage::W];
                unpack<T, Stage::W>(load<T, Stage::W>(stage.piece(q)), f);
#pragma unroll
                for (int i = 0; i < Stage::W; ++i) total += f[i] == NONE ? 0.f : expf(f[i] - top);
            }
        }
        if (nan) total = __uint_as_float(0x7fc00000u);
    }
    const float inverse = 1.f / total;
    for (int c0 = 0; c0 < a.experts; c0 += Stage::COLUMNS) {
        if (a.normalize) {
#pragma unroll
            for (int q = 0; q < 8; ++q) store<T, Stage::W>(stage.piece(q), Pack<T, Stage::W>{});
        } else {
            if (a.experts > Stage::COLUMNS) stage.fetch(logits, a.logits.stride, a.tokens - t0, c0, a.experts);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float f[Stage::W];
                unpack<T, Stage::W>(load<T, Stage::W>(stage.piece(q)), f);
#pragma unroll
                for (int i = 0; i < Stage::W; ++i) f[i] = f[i] == NONE ? 0.f : -(expf(f[i] - top) * inverse) * mean;
                store<T, Stage::W>(stage.piece(q), pack<T, Stage::W>(f));
            }
        }
#pragma unroll
        for (int j = 0; j < CHOSEN; ++j) {
            const int c = expert[j] - c0;
            if (expert[j] >= 0 && c >= 0 && c < Stage::COLUMNS) stage.piece(c / Stage::W)[c % Stage::W] = Element<T>::from(weight[j] * (grad[j] - mean));
        }
        stage.put(out, a.gradLogits.stride, a.tokens - t0, c0, a.experts);
    }
}

__global__ void __launch_bounds__(PARTITION_THREADS) route_place_kernel(const __grid_constant__ RouteArgs a, int tokensPerTile, const int* __restrict__ tileBefore,
                                                                        const int* __restrict__ totals)
{
    chained();
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
    placeSlots<TILE_ITEMS>(a, [&](int i) { return a.expert[firstSlot + i]; }, firstSlot, slots, start, counts);
}

template <class T, int LANES, int PER, bool VECTOR>
__global__ void __launch_bounds__(256) route_adjoint_kernel(const __grid_constant__ RouteArgs a)
{
    chained();
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
        using K = Key<T>;
        T raw[PER];
        loadLogits<T, PER, VECTOR>(static_cast<const T*>(a.logits.data) + row * a.logits.stride, lane, a.experts, raw);
        typename K::Type best = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const typename K::Type key = K::of(raw[i], lane * PER + i);
            best = key > best ? key : best;
        }
        best = groupMax<LANES>(best);
        const float top = K::value(best);
        float s = 0.f, z[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            z[i] = Element<T>::to(raw[i]);
            z[i] = best == 0 || z[i] == __uint_as_float(0xff800000u) ? 0.f : expf(z[i] - top);
            s += z[i];
        }
        const float inverse = 1.f / groupSum<LANES>(s);
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] = Element<T>::to(raw[i]) == __uint_as_float(0xff800000u) ? 0.f : -(z[i] * inverse) * mean;
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
// As in the embedding: a thread takes one access' worth of several rows, `pass` rows apart, so that it divides once; rows of more than 256 accesses are
// cut over blockIdx.y.
struct Place {
    int row, c;   // row within a block's first pass, element within the row
    bool inside;
    __device__ __forceinline__ Place(int perRow, int pass, int vec)
    {
        row = pass == 1 ? 0 : static_cast<int>(threadIdx.x) / perRow;
        const int access = pass == 1 ? blockIdx.y * 256 + threadIdx.x : threadIdx.x - row * perRow;
        inside = row < pass && access < perRow;
        c = access * vec;
    }
};

// rows[r] = x[order[r] / chosen], zeros behind the last expert's rows. 262144 rows of 256 half: 38 us, 5.4 TB/s (blocks that walk on: 41 us).
constexpr int MOVES = 4;
template <class T, int VEC>
__global__ void __launch_bounds__(256) dispatch_kernel(const __grid_constant__ ExchangeArgs a, int perRow, int pass)
{
    chained();
    constexpr int N = MOVES;
    const Place at(perRow, pass, VEC);
    if (!at.inside) return;
    const T* x = static_cast<const T*>(a.x.data);
    T* rows = static_cast<T*>(a.rows.data);
    const long long first = static_cast<long long>(blockIdx.x) * (pass * N) + at.row, slots = a.tokens * a.chosen;
    int token[N];
    Pack<T, VEC> v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int slot = first + k * pass < slots ? a.order[first + k * pass] : -1;
        token[k] = slot < 0 ? -1 : slot / a.chosen;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = {};
        if (token[k] >= 0 && token[k] < a.tokens) v[k] = load<T, VEC>(x + token[k] * a.x.stride + at.c);
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (first + k * pass < slots) store<T, VEC>(rows + (first + k * pass) * a.rows.stride + at.c, v[k]);
}

// x[t] = sum over the row's slots of (weight *) rows[position]. TOKENS rows per thread, SLOTS of each at a time; the blocks walk on with the list entries
// of their next rows fetched ahead (a row's load would wait for them else: 131072 rows of 256 half, 2 slots each, 48 -> 42 us weighted,
// 43 -> 34 to 39 us not).
template <class T, int VEC, bool WEIGHTED, int TOKENS, int SLOTS>
__global__ void __launch_bounds__(256) gather_sum_kernel(const __grid_constant__ ExchangeArgs a, Rows rowsIn, Rows out, int perRow, int pass)
{
    chained();
    const Place at(perRow, pass, VEC);
    if (!at.inside) return;
    const T* rows = static_cast<const T*>(rowsIn.data);
    const long long slots = a.tokens * a.chosen, step = static_cast<long long>(gridDim.x) * (pass * TOKENS);
    int nextPosition[TOKENS][SLOTS];
    float nextWeight[TOKENS][SLOTS];
    auto fetch = [&](long long first, int j0) {
#pragma unroll
        for (int k = 0; k < TOKENS; ++k)
#pragma unroll
            for (int j = 0; j < SLOTS; ++j) {
                const long long t = first + k * pass;
                nextPosition[k][j] = -1;
                nextWeight[k][j] = 1.f;
                if (t < a.tokens && j0 + j < a.chosen) {
                    nextPosition[k][j] = a.position[t * a.chosen + j0 + j];
                    if (WEIGHTED) nextWeight[k][j] = a.weights[t * a.chosen + j0 + j];
                }
            }
    };
    long long first = static_cast<long long>(blockIdx.x) * (pass * TOKENS) + at.row;
    fetch(first, 0);
    for (; first < a.tokens; first += step) {
        float2 sum[TOKENS][PAIRS<VEC>] = {};
        for (int j0 = 0; j0 < a.chosen; j0 += SLOTS) {
            float w[TOKENS][SLOTS];
            bool use[TOKENS][SLOTS];
            Pack<T, VEC> v[TOKENS][SLOTS];
#pragma unroll
            for (int k = 0; k < TOKENS; ++k)
#pragma unroll
                for (int j = 0; j < SLOTS; ++j) {
                    w[k][j] = nextWeight[k][j];
                    use[k][j] = nextPosition[k][j] >= 0 && nextPosition[k][j] < slots;
                    if (use[k][j]) v[k][j] = load<T, VEC>(rows + nextPosition[k][j] * rowsIn.stride + at.c);
                }
            if (j0 + SLOTS < a.chosen) fetch(first, j0 + SLOTS);
            else fetch(first + step, 0);
#pragma unroll
            for (int k = 0; k < TOKENS; ++k)
#pragma unroll
                for (int j = 0; j < SLOTS; ++j) {
                    if (!use[k][j]) continue;
                    float2 f[PAIRS<VEC>];
                    unpackPairs<T, VEC>(v[k][j], f);
#pragma unroll
                    for (int i = 0; i < PAIRS<VEC>; ++i) sum[k][i] = WEIGHTED ? fma2(both(w[k][j]), f[i], sum[k][i]) : add2(sum[k][i], f[i]);
                }
        }
#pragma unroll
        for (int k = 0; k < TOKENS; ++k)
            if (first + k * pass < a.tokens) store<T, VEC>(static_cast<T*>(out.data) + (first + k * pass) * out.stride + at.c, packPairs<T, VEC>(sum[k]));
    }
}

// Gradients of the combination: G lanes per row read its gradient, write the rows of gradients of SLOTS of its slots and add up their products with
// its rows. The rows without a slot, behind the last expert's, become zeros: row r is looked after by the lanes of row r / chosen.
template <class T, int VEC, int G, int SLOTS>
__global__ void __launch_bounds__(256, SLOTS <= 2 ? 5 : 3) combine_adjoint_kernel(const __grid_constant__ ExchangeArgs a)
{
    chained();
    const int lane = threadIdx.x % G;
    const long long slots = a.tokens * a.chosen, step = static_cast<long long>(gridDim.x) * (256 / G);
    const T* rows = static_cast<const T*>(a.rows.data);
    T* out = static_cast<T*>(a.gradRows.data);
    int nextPosition[SLOTS], nextOrder[SLOTS];
    float nextWeight[SLOTS];
    auto fetch = [&](long long t, int j0) {
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
            const long long s = t * a.chosen + j0 + j;
            const bool have = t < a.tokens && j0 + j < a.chosen;
            nextPosition[j] = have ? a.position[s] : -1;
            nextWeight[j] = have ? a.weights[s] : 0.f;
            nextOrder[j] = have && out != nullptr ? a.order[s] : 0;
        }
    };
    long long t = static_cast<long long>(blockIdx.x) * (256 / G) + threadIdx.x / G;
    fetch(t, 0);
    for (; t - threadIdx.x / G < a.tokens; t += step) {
        const bool active = t < a.tokens;
        const T* dy = static_cast<const T*>(a.gradX.data) + (active ? t : 0) * a.gradX.stride;
        for (int j0 = 0; j0 < a.chosen; j0 += SLOTS) {
            int position[SLOTS], order[SLOTS];
            float w[SLOTS];
            float2 dot[SLOTS] = {};
#pragma unroll
            for (int j = 0; j < SLOTS; ++j) {
                position[j] = nextPosition[j] < slots ? nextPosition[j] : -1;
                order[j] = nextOrder[j];
                w[j] = nextWeight[j];
            }
            bool fetched = false;
            if (active) {
                for (int c = lane * VEC; c < a.channels; c += G * VEC) {
                    const Pack<T, VEC> p = load<T, VEC>(dy + c);
                    Pack<T, VEC> v[SLOTS];
                    if (a.gradWeights != nullptr) {
#pragma unroll
                        for (int j = 0; j < SLOTS; ++j)
                            if (position[j] >= 0) v[j] = load<T, VEC>(rows + position[j] * a.rows.stride + c);
                    }
                    if (!fetched) {   // behind the first loads
                        fetched = true;
                        if (j0 + SLOTS < a.chosen) fetch(t, j0 + SLOTS);
                        else fetch(t + step, 0);
                    }
                    float2 g[PAIRS<VEC>];
                    unpackPairs<T, VEC>(p, g);
#pragma unroll
                    for (int j = 0; j < SLOTS; ++j) {
                        float2 f[PAIRS<VEC>];
                        if (out != nullptr && order[j] < 0) store<T, VEC>(out + (t * a.chosen + j0 + j) * a.gradRows.stride + c, Pack<T, VEC>{});
                        if (position[j] < 0) continue;
                        if (a.gradWeights != nullptr) {
                            unpackPairs<T, VEC>(v[j], f);
#pragma unroll
                            for (int k = 0; k < PAIRS<VEC>; ++k) dot[j] = fma2(g[k], f[k], dot[j]);
                        }
                        if (out != nullptr) {
#pragma unroll
                            for (int k = 0; k < PAIRS<VEC>; ++k) f[k] = mul2(both(w[j]), g[k]);
                            store<T, VEC>(out + position[j] * a.gradRows.stride + c, packPairs<T, VEC>(f));
                        }
                    }
                }
            }
            if (!fetched) {   // (lanes without a channel)
                if (j0 + SLOTS < a.chosen) fetch(t, j0 + SLOTS);
                else fetch(t + step, 0);
            }
            if (a.gradWeights == nullptr) continue;
#pragma unroll
            for (int j = 0; j < SLOTS; ++j) {
                const float all = groupSum<G>(dot[j].x + dot[j].y);
                if (active && lane == 0 && j0 + j < a.chosen) a.gradWeights[t * a.chosen + j0 + j] = all;
            }
        }
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

// A thread per row. Measured against groups of lanes, us: choice of 2 of 64 experts for 131072 rows of half 18 / 24, of 4 of 64 24 / 27, of 4 of 256 87 / 104,
// of 8 of 64 49 / 38 (the keys' order costs more than the groups' rounds), of 2 of 8 15 / 5 (groups of one lane); of 1 and 2 of 64 floats, whose keys have 64
// bits, 26 / 28 and 31 / 31, of 4 55 / 39. Adjoint, the mean of either kind of weights, 2 of 64 13 / 16, 8 of 256 48 / 75, 2 of 8 9 / 4; for 8192 rows 2 of 64
// 6 / 3.
static bool chooseByThread(const RouteArgs& a)
{
    return a.tokens >= 16384 && a.experts >= 32 && a.experts <= ROWS_EXPERTS && a.chosen <= (a.type == TYPE_FLOAT ? 2 : 4);
}
static bool adjointByThread(const RouteArgs& a) { return a.tokens >= 65536 && a.experts >= 32 && a.experts <= ROWS_EXPERTS && a.chosen <= ROWS_CHOSEN; }
template <class F>
static cudaError_t byChosen(int chosen, F&& f)
{
    if (chosen == 1) return f(std::integral_constant<int, 1>());
    if (chosen == 2) return f(std::integral_constant<int, 2>());
    if (chosen <= 4) return f(std::integral_constant<int, 4>());
    return f(std::integral_constant<int, 8>());
}

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
        if (!alone && vec && chooseByThread(a)) {
            auto go = [&](auto* kernel) {
                launchChained(kernel, p.tiles, 256, 32 * 1024, stream, 1, a, p.tokensPerTile, counts, p.tiles);
                return cudaGetLastError();
            };
            if (a.chosen == 1) return go(route_rows_kernel<T, 1>);
            if constexpr (sizeof(T) == 2) {
                if (a.chosen > 2) return go(route_rows_kernel<T, 4>);
            }
            return go(route_rows_kernel<T, 2>);
        }
        return byExperts(a.experts, [&](auto l, auto per) {
            constexpr int LANES = decltype(l)::value, PER = decltype(per)::value;
            const size_t bytes = (3 * (alone ? ALONE_SLOTS : TILE_SLOTS) + a.experts * (alone ? 1 + PARTITION_WARPS / 2 : 1)) * sizeof(int);
            auto go = [&](auto kernel) {
                launchChained(kernel, p.tiles, 256, bytes, stream, 1, a, p.tokensPerTile, counts, p.tiles);
                return cudaGetLastError();
            };
            if (vec) return alone ? go(route_choose_kernel<T, LANES, PER, true, true>) : go(route_choose_kernel<T, LANES, PER, true, false>);
            return alone ? go(route_choose_kernel<T, LANES, PER, false, true>) : go(route_choose_kernel<T, LANES, PER, false, false>);
        });
    });
    if (e != cudaSuccess || alone) return e;
    launchChained(partition_scan_kernel, a.experts, PARTITION_THREADS, 0, stream, 1, counts, before, totals, a.experts, p.tiles);
    launchChained(route_place_kernel, p.tiles, PARTITION_THREADS, (1 + PARTITION_WARPS / 2) * a.experts * sizeof(int), stream, 1, a, p.tokensPerTile, before, totals);
    return cudaGetLastError();
}

cudaError_t launchRouteAdjoint(const RouteArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    const bool vec = wide(a.logits, a.type, a.experts) && wide(a.gradLogits, a.type, a.experts);
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        if (vec && adjointByThread(a))
            return byChosen(a.chosen, [&](auto n) {
                launchChained(route_rows_adjoint_kernel<T, decltype(n)::value>, static_cast<unsigned>((a.tokens + 255) / 256), 256, 32 * 1024, stream, 1, a);
                return cudaGetLastError();
            });
        return byExperts(a.experts, [&](auto l, auto per) {
            constexpr int LANES = decltype(l)::value, PER = decltype(per)::value;
            const unsigned blocks = static_cast<unsigned>((a.tokens + 256 / LANES - 1) / (256 / LANES));
            if (vec) launchChained(route_adjoint_kernel<T, LANES, PER, true>, blocks, 256, 0, stream, 1, a);
            else launchChained(route_adjoint_kernel<T, LANES, PER, false>, blocks, 256, 0, stream, 1, a);
            return cudaGetLastError();
        });
    });
}

// grid of the kernels that walk accesses: `rows` rows, `each` of them per thread
struct AccessGrid {
    int perRow, pass;
    dim3 blocks;
    // walkers: at most this many blocks, which walk on
    AccessGrid(long long rows, int channels, int vec, int each, long long walkers = 1ll << 31)
    {
        perRow = channels / vec;
        pass = perRow > 128 ? 1 : 256 / perRow;
        const int parts = pass == 1 ? (perRow + 255) / 256 : 1;
        const long long all = (rows + pass * each - 1) / (pass * each), most = std::max(1ll, walkers / parts);
        blocks = dim3(static_cast<unsigned>(std::min(all, most)), parts);
    }
};

cudaError_t launchDispatch(const ExchangeArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        return byAccess<T>({&a.x, &a.rows}, a.type, a.channels, [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            const AccessGrid g(a.tokens * a.chosen, a.channels, VEC, MOVES);
            launchChained(dispatch_kernel<T, VEC>, g.blocks, 256, 0, stream, 1, a, g.perRow, g.pass);
            return cudaGetLastError();
        });
    });
}

template <class T, int VEC, bool WEIGHTED>
static cudaError_t launchGather(const ExchangeArgs& a, const Rows& in, const Rows& out, cudaStream_t stream)
{
    auto go = [&](auto* kernel, int each) {
        const AccessGrid g(a.tokens, a.channels, VEC, each, a.numSMs * 8ll);
        launchChained(kernel, g.blocks, 256, 0, stream, 1, a, in, out, g.perRow, g.pass);
        return cudaGetLastError();
    };
    // about 4 loads on their way per thread
    if (a.chosen == 1) return go(gather_sum_kernel<T, VEC, WEIGHTED, 4, 1>, 4);
    if (a.chosen == 2) return go(gather_sum_kernel<T, VEC, WEIGHTED, 2, 2>, 2);
    return go(gather_sum_kernel<T, VEC, WEIGHTED, 1, 4>, 1);
}
static cudaError_t launchGatherSum(const ExchangeArgs& a, const Rows& in, const Rows& out, bool weighted, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        return byAccess<T>({&in, &out}, a.type, a.channels, [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            return weighted ? launchGather<T, VEC, true>(a, in, out, stream) : launchGather<T, VEC, false>(a, in, out, stream);
        });
    });
}
cudaError_t launchDispatchAdjoint(const ExchangeArgs& a, cudaStream_t stream) { return launchGatherSum(a, a.gradRows, a.gradX, false, stream); }
cudaError_t launchCombine(const ExchangeArgs& a, cudaStream_t stream) { return launchGatherSum(a, a.rows, a.x, true, stream); }

cudaError_t launchCombineAdjoint(const ExchangeArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto v, auto g) {
            constexpr int VEC = decltype(v)::value, G = decltype(g)::value;
            const unsigned blocks = static_cast<unsigned>(std::min<long long>((a.tokens + 256 / G - 1) / (256 / G), a.numSMs * 8));
            if (a.chosen == 1) launchChained(combine_adjoint_kernel<T, VEC, G, 1>, blocks, 256, 0, stream, 1, a);
            else if (a.chosen == 2) launchChained(combine_adjoint_kernel<T, VEC, G, 2>, blocks, 256, 0, stream, 1, a);
            else launchChained(combine_adjoint_kernel<T, VEC, G, 4>, blocks, 256, 0, stream, 1, a);
            return cudaGetLastError();
        };
        return byAccess<T>({&a.rows, &a.gradX, &a.gradRows}, a.type, a.channels, [&](auto v) {
            return a.channels <= 8 * decltype(v)::value ? go(v, std::integral_constant<int, 8>()) : go(v, std::integral_constant<int, 32>());
        });
    });
}

} // namespace kernel
} // namespace qmlp
