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
// A thread takes one access' worth of LOOKUPS rows, `pass` rows apart, so that it divides once; 256 / accesses of a row rows per pass (rows of more than
// 256 accesses: blockIdx.y counts their parts).
constexpr int LOOKUPS = 4;
template <class T, int VEC>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const __grid_constant__ EmbeddingArgs a, int perRow, int pass)
{
    chained();
    constexpr int N = LOOKUPS;
    const T* table = static_cast<const T*>(a.table.data);
    T* y = static_cast<T*>(a.y.data);
    const int rowInPass = pass == 1 ? 0 : static_cast<int>(threadIdx.x) / perRow, access = blockIdx.y * 256 + (pass == 1 ? threadIdx.x : threadIdx.x - rowInPass * perRow);
    if (rowInPass >= pass || access >= perRow) return;
    const int c = access * VEC;
    const long long first = static_cast<long long>(blockIdx.x) * (pass * N) + rowInPass;
    long long token[N];
    Pack<T, VEC> v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) token[k] = first + k * pass < a.tokens ? tokenAt(a, first + k * pass) : -1;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = {};
        if (token[k] >= 0 && token[k] < a.rows) v[k] = load<T, VEC>(table + token[k] * a.table.stride + c);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (first + k * pass >= a.tokens) break;
        if (a.scale != 1.f && token[k] >= 0 && token[k] < a.rows) {   // (zeros stay zeros, whatever the scale)
            float f[VEC];
            unpack<T, VEC>(v[k], f);
#pragma unroll
            for (int i = 0; i < VEC; ++i) f[i] *= a.scale;
            v[k] = pack<T, VEC>(f);
        }
        store<T, VEC>(y + (first + k * pass) * a.y.stride + c, v[k]);
    }
}

// ---- sort -------------------------------------------------------------------------------------------------------------
// Tiles of 1024 tokens (256 threads) while they leave SMs without one, of 4096 (512 threads) above: the counters of a tile's digits are cleared and
// added up once per tile. A million tokens, 1024 digits, tiles of 2048 (256 threads): move 29 us; of 4096: 21 us.
// A tile's items go through shared memory into the order of their digits, so that what is written to memory lies side by side.
struct SortArgs {
    const int2* in;                // key and slot; null in the first pass: the tokens, and their own numbers
    int2* out;
    int *counts, *before, *totals;
    uint8_t* present;              // rows of the table that have a token, set in the last of several passes; null: another pass, or totals say so
    int items, blocks, shift, digits;
};
__device__ __forceinline__ int2 sortItem(const EmbeddingArgs& a, const SortArgs& s, int i)
{
    if (s.in != nullptr) return s.in[i];
    const long long r = tokenAt(a, i);
    return make_int2(static_cast<int>(r >= 0 && r < a.rows ? r : a.rows), i);
}
template <int ITEMS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) sort_count_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ SortArgs s)
{
    chained();
    __shared__ int count[PARTITION_MAX_DIGITS];
    for (int i = threadIdx.x; i < s.digits; i += WARPS * 32) count[i] = 0;
    const int first = blockIdx.x * (ITEMS * WARPS * 32);
    int key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = first + k * WARPS * 32 + threadIdx.x;
        key[k] = i < s.items ? sortItem(a, s, i).x : -1;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (key[k] >= 0) atomicAdd(&count[(key[k] >> s.shift) & (s.digits - 1)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < s.digits; i += WARPS * 32) s.counts[static_cast<long long>(i) * s.blocks + blockIdx.x] = count[i];
}
template <int ITEMS, int WARPS>
constexpr int moveBytes(int digits) { return ITEMS * WARPS * 32 * 8 + 2 * digits * 4 + WARPS * digits * 2; }
template <int ITEMS, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1024 / (WARPS * 32)) sort_move_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ SortArgs s)
{
    chained();
    constexpr int THREADS = WARPS * 32, TILE = ITEMS * THREADS;
    extern __shared__ __align__(16) int2 sorted[];                           // TILE
    int *start = reinterpret_cast<int*>(sorted + TILE), *local = start + s.digits;   // digits: where the tile's items go, in memory and in the tile
    uint16_t* counts = reinterpret_cast<uint16_t*>(local + s.digits);        // warps x digits
    __shared__ int warpSums[WARPS];
    for (int i = threadIdx.x; i < s.digits; i += THREADS) start[i] = s.totals[i];
    __syncthreads();
    blockExclusive<WARPS>(start, s.digits, warpSums);
    const int first = blockIdx.x * TILE;
    for (int d = threadIdx.x; d < s.digits; d += THREADS) start[d] += s.before[static_cast<long long>(blockIdx.x) * s.digits + d];
    int digit[ITEMS], rank[ITEMS];
    tileRanks<ITEMS, WARPS>([&](int i) { return first + i < s.items ? (sortItem(a, s, first + i).x >> s.shift) & (s.digits - 1) : -1; }, s.digits, counts, digit, rank);
    for (int d = threadIdx.x; d < s.digits; d += THREADS) local[d] = warpOffsets<WARPS>(counts, s.digits, d);
    __syncthreads();
    blockExclusive<WARPS>(local, s.digits, warpSums);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)   // (the items once more: they would cost the registers of a second block)
        if (digit[k] >= 0) sorted[local[digit[k]] + counts[warp * s.digits + digit[k]] + rank[k]] = sortItem(a, s, first + (warp * ITEMS + k) * 32 + lane);
    __syncthreads();
    const int here = min(TILE, s.items - first);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = k * THREADS + threadIdx.x;
        if (i >= here) break;
        const int2 v = sorted[i];
        const int d = (v.x >> s.shift) & (s.digits - 1);
        s.out[start[d] + i - local[d]] = v;
        // (sorted by now within the tile: once per row and tile. By the count of the first digit, per warp, a table of 1985 rows cost 97 us, not 15:
        // stores to the same few lines wait for one another)
        if (s.present != nullptr && v.x < a.rows && (i == 0 || sorted[i - 1].x != v.x)) s.present[v.x] = 1;
    }
}

// ---- sums over runs of equal tokens -------------------------------------------------------------------------------------
struct RunArgs {
    const int2* sorted;            // key, slot
    const uint8_t* present;        // rows with a token, or null:
    const int* totals;             // tokens of a row
    int items, chunk, chunks, runBlocks;
    float* partial;      // chunks x 2 x channels: the run a chunk begins with (if it began before), the run it ends with (if it goes on)
};
constexpr int RUN_STEP = 8;    // rows in flight per group; chunks are multiples of it
constexpr int FILL_ROWS = 8;   // rows of the table a group looks at

// Blocks of the first kind add up runs, a chunk per group of G lanes; the others write the zeros of the rows without a token meanwhile.
template <class T, int VEC, int G>
__global__ void __launch_bounds__(256, 3) embedding_runs_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ RunArgs r)
{
    chained();
    constexpr int GROUPS = 256 / G;
    const int c = (blockIdx.y * G + threadIdx.x % G) * VEC;
    if (c >= a.channels) return;
    T* out = static_cast<T*>(a.gradTable.data);
    if (blockIdx.x >= static_cast<unsigned>(r.runBlocks)) {
        const long long first = (static_cast<long long>(blockIdx.x - r.runBlocks) * FILL_ROWS) * GROUPS + threadIdx.x / G;
#pragma unroll
        for (int k = 0; k < FILL_ROWS; ++k) {
            const long long row = first + k * GROUPS;
            if (row < a.rows && (r.present != nullptr ? r.present[row] == 0 : r.totals[row] == 0)) store<T, VEC>(out + row * a.gradTable.stride + c, Pack<T, VEC>{});
        }
        return;
    }
    const int chunk = blockIdx.x * GROUPS + threadIdx.x / G;
    if (chunk >= r.chunks) return;
    const T* dy = static_cast<const T*>(a.gradY.data);
    const int begin = chunk * r.chunk, end = min(r.items, begin + r.chunk);
    const int none = static_cast<int>(a.rows);   // key of the tokens outside the table
    int current = r.sorted[begin].x;
    bool entered = begin > 0 && r.sorted[begin - 1].x == current;   // the current run began in an earlier chunk
    float sum[VEC] = {};
    auto flush = [&](bool leaves) {
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
    };
    // the list holds whole steps (behind the last item: whatever, not used), 16-byte aligned
    int4 next[RUN_STEP / 2];
    auto fetch = [&](int i) {
#pragma unroll
        for (int h = 0; h < RUN_STEP / 2; ++h) next[h] = *reinterpret_cast<const int4*>(r.sorted + i + 2 * h);
    };
    fetch(begin);
    for (int i = begin; i < end; i += RUN_STEP) {
        int key[RUN_STEP], slot[RUN_STEP];
#pragma unroll
        for (int h = 0; h < RUN_STEP / 2; ++h) {
            key[2 * h] = next[h].x;
            slot[2 * h] = next[h].y;
            key[2 * h + 1] = next[h].z;
            slot[2 * h + 1] = next[h].w;
        }
        if (i + RUN_STEP < end) fetch(i + RUN_STEP);
        Pack<T, VEC> v[RUN_STEP];
#pragma unroll
        for (int k = 0; k < RUN_STEP; ++k) {
            if (i + k >= end) key[k] = none;
            v[k] = {};
            if (key[k] < none) v[k] = load<T, VEC>(dy + static_cast<long long>(slot[k]) * a.gradY.stride + c);
        }
        if (key[0] == current && key[RUN_STEP - 1] == current && current < none) {   // one run
#pragma unroll
            for (int k = 0; k < RUN_STEP; ++k) {
                float f[VEC];
                unpack<T, VEC>(v[k], f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += f[j];
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < RUN_STEP; ++k) {
            if (i + k >= end) break;
            if (key[k] != current) {
                if (current < none) flush(false);
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
    if (current < none) flush(end < r.items && r.sorted[end].x == current);
}

// Joins the runs that cross chunks. A block looks at JOIN_CHUNKS chunks, a warp each; for every run that begins in one of them and goes on behind
// it, its parts are added up: by G lanes side by side along the columns where they are few, else by 512 / G such shares of
// consecutive parts, then the shares in order.
constexpr int JOIN_CHUNKS = 8, JOIN_FEW = 16;
template <class T, int G>
__global__ void __launch_bounds__(512) embedding_join_kernel(const __grid_constant__ EmbeddingArgs a, const __grid_constant__ RunArgs r)
{
    chained();
    constexpr int SHARES = 512 / G;
    __shared__ int keyOf[JOIN_CHUNKS], partsOf[JOIN_CHUNKS];
    __shared__ float shared[512];
    if (threadIdx.x < JOIN_CHUNKS * 32) {   // a warp per chunk
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int chunk = blockIdx.x * JOIN_CHUNKS + warp, begin = chunk * r.chunk, end = begin + r.chunk;
        int parts = 0, key = 0;
        if (chunk < r.chunks && end < r.items) {
            key = r.sorted[end].x;
            const int last = r.sorted[end - 1].x, first = r.sorted[begin].x, before = begin > 0 ? r.sorted[begin - 1].x : -1;
            if (key < static_cast<int>(a.rows) && last == key && !(first == key && before == key)) {
                // the tail of `chunk`, and the heads of the chunks whose first item still has the key: 32 looked at in a step, the steps 32 times
                // as long for as long as all have it
                int known = chunk + 1;   // has it
                for (int stride = 1;;) {
                    const long long probe = known + static_cast<long long>(lane + 1) * stride;
                    const unsigned have = __ballot_sync(0xffffffffu, probe < r.chunks && r.sorted[probe * r.chunk].x == key);
                    known += __popc(have) * stride;
                    if (have == 0xffffffffu) {
                        if (stride <= 1024) stride *= 32;
                    } else if (stride == 1) {
                        break;
                    } else {
                        stride /= 32;
                    }
                }
                parts = known + 1 - chunk;
            }
        }
        if (lane == 0) {
            keyOf[warp] = key;
            partsOf[warp] = parts;
        }
    }
    __syncthreads();
    const int share = threadIdx.x / G, c = blockIdx.y * G + threadIdx.x % G;
    const long long pair = 2ll * a.channels;
    const float* from = r.partial + static_cast<long long>(blockIdx.x) * JOIN_CHUNKS * pair + c;
    auto write = [&](int k, float sum) {
        static_cast<T*>(a.gradTable.data)[static_cast<long long>(keyOf[k]) * a.gradTable.stride + c] = Element<T>::from(sum * a.scale);
    };
    // runs of few parts: a share each
    for (int k = share; k < JOIN_CHUNKS; k += SHARES) {
        const int parts = partsOf[k];
        if (parts == 0 || parts > JOIN_FEW || c >= a.channels) continue;
        float v[JOIN_FEW], sum = 0.f;
#pragma unroll
        for (int p = 0; p < JOIN_FEW; ++p) v[p] = p < parts ? from[(k + p) * pair + (p == 0 ? a.channels : 0)] : 0.f;
#pragma unroll
        for (int p = 0; p < JOIN_FEW; ++p) sum += v[p];
        write(k, sum);
    }
    for (int k = 0; k < JOIN_CHUNKS; ++k) {
        const int parts = partsOf[k];
        if (parts <= JOIN_FEW) continue;
        const int each = (parts + SHARES - 1) / SHARES, first = share * each, last = min(parts, first + each);
        float sum = 0.f;
        if (c < a.channels) {
#pragma unroll 8
            for (int p = first; p < last; ++p) sum += from[(k + p) * pair + (p == 0 ? a.channels : 0)];
        }
        shared[threadIdx.x] = sum;
        __syncthreads();
        if (share == 0 && c < a.channels) {
            const int used = (parts + each - 1) / each;
            for (int s = 1; s < used; ++s) sum += shared[s * G + threadIdx.x];
            write(k, sum);
        }
        __syncthreads();
    }
}

// ---- launch --------------------------------------------------------------------------------------------------------------
size_t align256(size_t b) { return (b + 255) / 256 * 256; }

struct SortPlan {
    int passes, bits, digits, blocks, chunk, chunks;
    bool large;
    size_t list, counts, before, totals, present, partial, bytes;   // bytes of one list of keys and slots, offsets of the rest
    SortPlan(long long tokens, long long rows, int channels, int type, int numSMs)
    {
        int keyBits = 1;
        while ((1ll << keyBits) < rows + 1) ++keyBits;
        passes = (keyBits + 9) / 10;
        bits = (keyBits + passes - 1) / passes;
        digits = 1 << bits;
        large = tokens > numSMs * 2048ll;
        const int tile = large ? 4096 : 1024;
        blocks = static_cast<int>((tokens + tile - 1) / tile);
        // chunks: 512 threads' worth of groups per SM, 8 rows in flight each (1024: sums 34 us and joins 10 us for a million rows of 32 floats, against 30 and 6)
        const int wide = 16 / typeBytes(type);
        const long long lanes = std::max<long long>(1, (channels + wide - 1) / wide), groups = std::max<long long>(1, numSMs * 512ll / lanes);
        chunk = static_cast<int>(std::min<long long>(256, std::max<long long>(16, (tokens + groups - 1) / groups)));
        chunk = (chunk + RUN_STEP - 1) / RUN_STEP * RUN_STEP;
        chunks = static_cast<int>((tokens + chunk - 1) / chunk);
        list = align256((static_cast<size_t>(tokens) + RUN_STEP) * sizeof(int2));
        counts = (passes > 1 ? 2 : 1) * list;
        before = counts + align256(static_cast<size_t>(digits) * blocks * 4);
        totals = before + align256(static_cast<size_t>(digits) * blocks * 4);
        present = totals + align256(digits * 4);
        partial = present + (passes > 1 ? align256(static_cast<size_t>(rows)) : 0);
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
template <class F>
cudaError_t byLanes(int vectors, F&& f)
{
    if (vectors <= 1) return f(std::integral_constant<int, 1>());
    if (vectors <= 4) return f(std::integral_constant<int, 4>());
    if (vectors <= 8) return f(std::integral_constant<int, 8>());
    if (vectors <= 16) return f(std::integral_constant<int, 16>());
    return f(std::integral_constant<int, 32>());
}
template <class T, int VEC>
cudaError_t launchRuns(const EmbeddingArgs& a, RunArgs r, cudaStream_t stream)
{
    const int vectors = (a.channels + VEC - 1) / VEC;
    return byLanes(vectors, [&](auto g) {
        constexpr int G = decltype(g)::value, GROUPS = 256 / G;
        r.runBlocks = (r.chunks + GROUPS - 1) / GROUPS;
        const long long fill = (a.rows + GROUPS * FILL_ROWS - 1) / (GROUPS * FILL_ROWS);
        launchChained(embedding_runs_kernel<T, VEC, G>, dim3(static_cast<unsigned>(r.runBlocks + fill), (vectors + G - 1) / G), 256, 0, stream, 1, a, r);
        return cudaGetLastError();
    });
}
template <int ITEMS, int WARPS>
cudaError_t launchSort(const EmbeddingArgs& a, const SortArgs& s, cudaStream_t stream)
{
    launchChained(sort_count_kernel<ITEMS, WARPS>, s.blocks, WARPS * 32, 0, stream, 1, a, s);
    launchChained(partition_scan_kernel, s.digits, PARTITION_THREADS, 0, stream, 1, s.counts, s.before, s.totals, s.digits, s.blocks);
    if (moveBytes<ITEMS, WARPS>(PARTITION_MAX_DIGITS) > 48 * 1024) {
        const cudaError_t e = allowShared(reinterpret_cast<const void*>(sort_move_kernel<ITEMS, WARPS>), moveBytes<ITEMS, WARPS>(PARTITION_MAX_DIGITS));
        if (e != cudaSuccess) return e;
    }
    launchChained(sort_move_kernel<ITEMS, WARPS>, s.blocks, WARPS * 32, moveBytes<ITEMS, WARPS>(s.digits), stream, 1, a, s);
    return cudaGetLastError();
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
        return byAccess<T>({&a.table, &a.y}, a.type, a.channels, [&](auto v) {
            constexpr int VEC = decltype(v)::value, N = LOOKUPS;
            const int perRow = a.channels / VEC, pass = perRow > 128 ? 1 : 256 / perRow;
            const dim3 grid(static_cast<unsigned>((a.tokens + pass * N - 1) / (pass * N)), pass == 1 ? (perRow + 255) / 256 : 1);
            launchChained(embedding_forward_kernel<T, VEC>, grid, 256, 0, stream, 1, a, perRow, pass);
            return cudaGetLastError();
        });
    });
}

cudaError_t launchEmbeddingAdjoint(const EmbeddingArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    if (a.tokens == 0)
        return cudaMemset2DAsync(a.gradTable.data, static_cast<size_t>(a.gradTable.stride) * typeBytes(a.type), 0, static_cast<size_t>(a.channels) * typeBytes(a.type),
                                 static_cast<size_t>(a.rows), stream);
    const SortPlan p(a.tokens, a.rows, a.channels, a.type, a.numSMs);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    int2* lists[2] = {reinterpret_cast<int2*>(base), reinterpret_cast<int2*>(base + p.list)};
    SortArgs s{};
    s.counts = reinterpret_cast<int*>(base + p.counts);
    s.before = reinterpret_cast<int*>(base + p.before);
    s.totals = reinterpret_cast<int*>(base + p.totals);
    uint8_t* present = p.passes > 1 ? base + p.present : nullptr;
    s.items = static_cast<int>(a.tokens);
    s.blocks = p.blocks;
    s.digits = p.digits;
    cudaError_t e = p.passes > 1 ? cudaMemsetAsync(present, 0, static_cast<size_t>(a.rows), stream) : cudaSuccess;
    for (int k = 0; k < p.passes && e == cudaSuccess; ++k) {
        s.in = k > 0 ? lists[(k + 1) & 1] : nullptr;
        s.out = lists[k & 1];
        s.shift = k * p.bits;
        s.present = k == p.passes - 1 ? present : nullptr;
        e = p.large ? launchSort<8, 16>(a, s, stream) : launchSort<4, 8>(a, s, stream);
    }
    if (e != cudaSuccess) return e;
    RunArgs r{s.out, present, s.totals, s.items, p.chunk, p.chunks, 0, reinterpret_cast<float*>(base + p.partial)};
    return byType(a.type, [&](auto t) {
        using T = decltype(t);
        const cudaError_t status = byAccess<T>({&a.gradTable, &a.gradY}, a.type, a.channels, [&](auto v) { return launchRuns<T, decltype(v)::value>(a, r, stream); });
        if (status != cudaSuccess || p.chunks < 2) return status;
        return byLanes(a.channels, [&](auto g) {
            constexpr int G = decltype(g)::value;
            launchChained(embedding_join_kernel<T, G>, dim3((p.chunks + JOIN_CHUNKS - 1) / JOIN_CHUNKS, (a.channels + G - 1) / G), 512, 0, stream, 1, a, r);
            return cudaGetLastError();
        });
    });
}

} // namespace kernel
} // namespace qmlp
