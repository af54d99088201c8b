// Embedding lookup with a scale, and the gradient of its table.
//
//   y_t = scale * table[token_t]          (a row of zeros where token_t lies outside the table)
//   d table_v = scale * sum of dy_t over the tokens with token_t = v
//
// Forward: one 16-byte access per thread and step, rows of the table come from L2 where tokens repeat.
// Gradient: the tokens are sorted (stable, radix of up to 10 bits per pass; tokens outside the table go behind the last row),
// so that the occurrences of a row lie side by side in the order of the batch. A chunk of sorted occurrences belongs to a
// group of lanes, which adds up fp32 sums in registers and writes a row once, when the token changes. Runs that cross chunks
// leave partial sums that a second kernel joins, in order. No atomics: the result does not change from run to run, and hot rows
// cost no more than others. The rows without a token are zeros.
#include "partition.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

__device__ __forceinline__ long long tokenAt(const EmbeddingArgs& a, long long t)
{
    return a.tokenType == TYPE_INT64 ? static_cast<const long long*>(a.token)[t * a.tokenStride]
                                     : static_cast<long long>(static_cast<const int*>(a.token)[t * a.tokenStride]);
}

// ---- forward -----------------------------------------------------------------------------------------------------------
constexpr int LOOKUPS = 4;   // accesses in flight per thread
template <class T, int VEC>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const __grid_constant__ EmbeddingArgs a, long long total, int perRow)
{
    const T* table = static_cast<const T*>(a.table.data);
    T* y = static_cast<T*>(a.y.data);
    const long long first = blockIdx.x * (256ll * LOOKUPS) + threadIdx.x;
    Pack<T, VEC> v[LOOKUPS];
    long long at[LOOKUPS];
#pragma unroll
    for (int k = 0; k < LOOKUPS; ++k) {
        const long long i = first + k * 256;
        at[k] = -1;
        v[k] = {};
        if (i >= total) continue;
        const long long t = total <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(perRow) : i / perRow;
        const int c = static_cast<int>(i - t * perRow) * VEC;
        at[k] = t * a.y.stride + c;
        const long long r = tokenAt(a, t);
        if (r >= 0 && r < a.rows) v[k] = load<T, VEC>(table + r * a.table.stride + c);
    }
#pragma unroll
    for (int k = 0; k < LOOKUPS; ++k) {
        if (at[k] < 0) continue;
        if (a.scale != 1.f) {
            float f[VEC];
            unpack<T, VEC>(v[k], f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] *= a.scale;
            v[k] = pack<T, VEC>(f);
        }
        store<T, VEC>(y + at[k], v[k]);
    }
}

// ---- sort -------------------------------------------------------------------------------------------------------------
constexpr int SORT_ITEMS = 8, SORT_TILE = SORT_ITEMS * PARTITION_THREADS;

struct SortArgs {
    const int *keysIn, *slotsIn;   // null in the first pass: tokens, and their own numbers
    int *keysOut, *slotsOut;
    int *counts, *totals;
    int items, blocks, shift, digits;
};
__device__ __forceinline__ int sortKey(const EmbeddingArgs& a, const SortArgs& s, int i)
{
    if (s.keysIn != nullptr) return s.keysIn[i];
    const long long r = tokenAt(a, i);
    return static_cast<int>(r >= 0 && r < a.rows ? r : a.rows);
}
__global__ void __launch_bounds__(PARTITION_THREADS) sort_count_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ SortArgs s)
{
    __shared__ int count[PARTITION_MAX_DIGITS];
    for (int i = threadIdx.x; i < s.digits; i += PARTITION_THREADS) count[i] = 0;
    __syncthreads();
    const int first = blockIdx.x * SORT_TILE;
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; ++k) {
        const int i = first + k * PARTITION_THREADS + threadIdx.x;
        if (i < s.items) atomicAdd(&count[(sortKey(a, s, i) >> s.shift) & (s.digits - 1)], 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s.digits; i += PARTITION_THREADS) s.counts[static_cast<long long>(i) * s.blocks + blockIdx.x] = count[i];
}
__global__ void __launch_bounds__(PARTITION_THREADS) sort_move_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ SortArgs s)
{
    extern __shared__ int dynamic[];
    int *start = dynamic, *counts = dynamic + s.digits;   // digits, warps x digits
    __shared__ int warpSums[PARTITION_WARPS];
    for (int i = threadIdx.x; i < s.digits; i += PARTITION_THREADS) start[i] = s.totals[i];
    __syncthreads();
    blockExclusive(start, s.digits, warpSums);
    const int first = blockIdx.x * SORT_TILE;
    int digit[SORT_ITEMS], rank[SORT_ITEMS], key[SORT_ITEMS], at = 0;
    tileRanks<SORT_ITEMS>([&](int i) {
        const int k = first + i < s.items ? sortKey(a, s, first + i) : -1;
        key[at++] = k;
        return k < 0 ? -1 : (k >> s.shift) & (s.digits - 1);
    }, s.digits, counts, digit, rank);
    for (int d = threadIdx.x; d < s.digits; d += PARTITION_THREADS)
        warpOffsets(counts, s.digits, d, start[d] + s.counts[static_cast<long long>(d) * s.blocks + blockIdx.x]);
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < SORT_ITEMS; ++k) {
        if (digit[k] < 0) continue;
        const int i = first + (warp * SORT_ITEMS + k) * 32 + lane, to = counts[warp * s.digits + digit[k]] + rank[k];
        s.keysOut[to] = key[k];
        s.slotsOut[to] = s.slotsIn != nullptr ? s.slotsIn[i] : i;
    }
}

// ---- sums over runs of equal tokens -------------------------------------------------------------------------------------
struct RunArgs {
    const int *keys, *slots;
    int items, chunk, chunks;
    float* partial;      // chunks x 2 x channels: the run a chunk begins with (if it began before), the run it ends with (if it goes on)
};
constexpr int RUN_UNROLL = 4;

template <class T, int VEC, int G>
__global__ void __launch_bounds__(256) embedding_runs_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ RunArgs r)
{
    constexpr int GROUPS = 256 / G;
    const int chunk = blockIdx.x * GROUPS + threadIdx.x / G;
    const int c = (blockIdx.y * G + threadIdx.x % G) * VEC;
    if (chunk >= r.chunks || c >= a.channels) return;
    const T* dy = static_cast<const T*>(a.gradY.data);
    T* out = static_cast<T*>(a.gradTable.data);
    const int begin = chunk * r.chunk, end = min(r.items, begin + r.chunk);
    const int none = static_cast<int>(a.rows);   // key of the tokens outside the table
    int current = r.keys[begin];
    bool entered = begin > 0 && r.keys[begin - 1] == current;   // the current run began in an earlier chunk
    float sum[VEC] = {};
    auto flush = [&](bool leaves) {
        if (current < none) {
            if (!entered && !leaves) {
                float f[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[i] = sum[i] * a.scale;
                store<T, VEC>(out + static_cast<long long>(current) * a.gradTable.stride + c, pack<T, VEC>(f));
            } else {
                float* p = r.partial + (static_cast<long long>(chunk) * 2 + (entered ? 0 : 1)) * a.channels + c;
#pragma unroll
                for (int i = 0; i < VEC; ++i) p[i] = sum[i];
            }
        }
    };
    for (int i = begin; i < end; i += RUN_UNROLL) {
        int key[RUN_UNROLL];
        Pack<T, VEC> v[RUN_UNROLL];
#pragma unroll
        for (int k = 0; k < RUN_UNROLL; ++k) {
            key[k] = i + k < end ? r.keys[i + k] : none;
            if (key[k] < none) v[k] = load<T, VEC>(dy + static_cast<long long>(r.slots[i + k]) * a.gradY.stride + c);
        }
#pragma unroll
        for (int k = 0; k < RUN_UNROLL; ++k) {
            if (i + k >= end) break;
            if (key[k] != current) {
                flush(false);
                current = key[k];
                entered = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
            }
            if (current >= none) return;   // behind the last row of the table: nothing more to add
            float f[VEC];
            unpack<T, VEC>(v[k], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[j] += f[j];
        }
    }
    flush(end < r.items && r.keys[end] == current);
}

// A block per chunk: if a run begins in it and goes on behind it, the sums of its parts, in order: each of the block's 8 warps
// adds up consecutive parts, then the warps' sums follow one another.
template <class T>
__global__ void __launch_bounds__(256) embedding_join_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ RunArgs r)
{
    __shared__ float shared[8][32];
    const int chunk = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int end = (chunk + 1) * r.chunk;
    if (end >= r.items) return;
    const int key = r.keys[end];
    const int begin = chunk * r.chunk;
    if (key >= static_cast<int>(a.rows) || r.keys[end - 1] != key || (r.keys[begin] == key && begin > 0 && r.keys[begin - 1] == key)) return;
    // chunks whose first key is still `key`: the run enters them
    int low = chunk + 1, high = r.chunks;   // the run enters `low`, not `high`
    while (low + 1 < high) {
        const int mid = (low + high) / 2;
        if (r.keys[mid * r.chunk] == key) low = mid;
        else high = mid;
    }
    const int parts = low + 1 - chunk;      // the tail of `chunk`, the heads of chunk + 1 .. low
    const int share = (parts + 7) / 8, from = warp * share, to = min(parts, from + share);
    const int c = blockIdx.y * 32 + lane;
    float sum = 0.f;
    if (c < a.channels) {
#pragma unroll 8
        for (int p = from; p < to; ++p) sum += r.partial[(static_cast<long long>(chunk + p) * 2 + (p == 0 ? 1 : 0)) * a.channels + c];
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < a.channels) {
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += shared[w][lane];
        static_cast<T*>(a.gradTable.data)[static_cast<long long>(key) * a.gradTable.stride + c] = Element<T>::from(sum * a.scale);
    }
}

// ---- launch --------------------------------------------------------------------------------------------------------------
size_t align256(size_t b) { return (b + 255) / 256 * 256; }

struct SortPlan {
    int passes, bits, digits, blocks, chunk, chunks;
    size_t keys, counts, totals, partial, bytes;   // bytes of one array of keys, offsets of the rest
    SortPlan(long long tokens, long long rows, int channels, int type, int numSMs)
    {
        int keyBits = 1;
        while ((1ll << keyBits) < rows + 1) ++keyBits;
        passes = (keyBits + 9) / 10;
        bits = (keyBits + passes - 1) / passes;
        digits = 1 << bits;
        blocks = static_cast<int>((tokens + SORT_TILE - 1) / SORT_TILE);
        // chunks of 16 occurrences and more: enough of them that every SM has 32 warps' worth, one group of lanes each
        const long long lanes = std::max<long long>(1, (channels + 16 / typeBytes(type) - 1) / (16 / typeBytes(type)));
        const long long groups = std::max<long long>(1, static_cast<long long>(numSMs) * 1024 / lanes);
        chunk = static_cast<int>(std::min<long long>(256, std::max<long long>(16, (tokens + groups - 1) / groups)));
        chunks = static_cast<int>((tokens + chunk - 1) / chunk);
        keys = align256(static_cast<size_t>(tokens) * 4);
        counts = 4 * keys;
        totals = counts + align256(static_cast<size_t>(digits) * blocks * 4);
        partial = totals + align256(digits * 4);
        bytes = partial + align256(static_cast<size_t>(chunks) * 2 * channels * 4);
    }
};

template <class F>
cudaError_t byType(int type, F&& f)
{
    switch (type) {
    case TYPE_FLOAT: return f(float());
    case TYPE_HALF: return f(__half());
    default: return f(__nv_bfloat16());
    }
}
template <class T, int VEC>
cudaError_t launchRuns(const EmbeddingArgs& a, const RunArgs& r, cudaStream_t stream)
{
    const int vectors = (a.channels + VEC - 1) / VEC;
    auto go = [&](auto g) {
        constexpr int G = decltype(g)::value;
        embedding_runs_kernel<T, VEC, G><<<dim3((r.chunks + 256 / G - 1) / (256 / G), (vectors + G - 1) / G), 256, 0, stream>>>(a, r);
        return cudaGetLastError();
    };
    if (vectors <= 1) return go(std::integral_constant<int, 1>());
    if (vectors <= 4) return go(std::integral_constant<int, 4>());
    if (vectors <= 8) return go(std::integral_constant<int, 8>());
    if (vectors <= 16) return go(std::integral_constant<int, 16>());
    return go(std::integral_constant<int, 32>());
}

} // namespace

size_t embeddingAdjointBytes(long long tokens, long long rows, int channels, int type, int numSMs)
{
    return tokens == 0 ? 0 : SortPlan(tokens, rows, channels, type, numSMs).bytes;
}

cudaError_t launchEmbeddingForward(const EmbeddingArgs& a, cudaStream_t stream)
{
    if (a.tokens == 0) return cudaSuccess;
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = wide(a.table, a.type, a.channels) && wide(a.y, a.type, a.channels);
        const int perRow = vec ? a.channels / WIDE<T> : a.channels;
        const long long total = a.tokens * perRow, blocks = (total + 256 * LOOKUPS - 1) / (256 * LOOKUPS);
        if (vec) embedding_forward_kernel<T, WIDE<T>><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, total, perRow);
        else embedding_forward_kernel<T, 1><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a, total, perRow);
        return cudaGetLastError();
    });
}

cudaError_t launchEmbeddingAdjoint(const EmbeddingArgs& a, cudaStream_t stream)
{
    cudaError_t e = cudaSuccess;
    if (a.rows > 0)
        e = cudaMemset2DAsync(a.gradTable.data, static_cast<size_t>(a.gradTable.stride) * typeBytes(a.type), 0,
                              static_cast<size_t>(a.channels) * typeBytes(a.type), static_cast<size_t>(a.rows), stream);
    if (e != cudaSuccess || a.tokens == 0 || a.rows == 0) return e;
    const SortPlan p(a.tokens, a.rows, a.channels, a.type, a.numSMs);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    int* keys[2] = {reinterpret_cast<int*>(base), reinterpret_cast<int*>(base + p.keys)};
    int* slots[2] = {reinterpret_cast<int*>(base + 2 * p.keys), reinterpret_cast<int*>(base + 3 * p.keys)};
    SortArgs s{};
    s.counts = reinterpret_cast<int*>(base + p.counts);
    s.totals = reinterpret_cast<int*>(base + p.totals);
    s.items = static_cast<int>(a.tokens);
    s.blocks = p.blocks;
    s.digits = p.digits;
    for (int k = 0; k < p.passes; ++k) {
        s.keysIn = k > 0 ? keys[(k + 1) & 1] : nullptr;
        s.slotsIn = k > 0 ? slots[(k + 1) & 1] : nullptr;
        s.keysOut = keys[k & 1];
        s.slotsOut = slots[k & 1];
        s.shift = k * p.bits;
        sort_count_kernel<<<p.blocks, PARTITION_THREADS, 0, stream>>>(a, s);
        partition_scan_kernel<<<(p.digits + PARTITION_WARPS - 1) / PARTITION_WARPS, PARTITION_THREADS, 0, stream>>>(s.counts, s.totals, p.digits, p.blocks);
        sort_move_kernel<<<p.blocks, PARTITION_THREADS, (PARTITION_WARPS + 1) * p.digits * sizeof(int), stream>>>(a, s);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    RunArgs r{s.keysOut, s.slotsOut, s.items, p.chunk, p.chunks, reinterpret_cast<float*>(base + p.partial)};
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const bool vec = wide(a.gradTable, a.type, a.channels) && wide(a.gradY, a.type, a.channels);
        const cudaError_t status = vec ? launchRuns<T, WIDE<T>>(a, r, stream) : launchRuns<T, 1>(a, r, stream);
        if (status != cudaSuccess || p.chunks < 2) return status;
        embedding_join_kernel<T><<<dim3(p.chunks - 1, (a.channels + 31) / 32), 256, 0, stream>>>(a, r);
        return cudaGetLastError();
    });
}

} // namespace kernel
} // namespace qmlp
