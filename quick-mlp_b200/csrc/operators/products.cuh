// What the kernels of the products grouped by expert share (16-bit operands in expert_linear.cu, 4-bit ones in mx_linear.cu): the instructions of
// tensor cores, tensor memory and pairs of blocks, the plan of the experts' tiles, bounded waits, the store of a tile.
#pragma once
#include "common.cuh"

#include <type_traits>

#include <cuda.h>

namespace qmlp {
namespace kernel {
namespace products {

using namespace ops;

// ---- PTX ---------------------------------------------------------------------------------------------------------------
// ---- pairs of blocks: the leader (rank 0) issues the products of both, its barriers are reached from the other by their cluster address
__device__ __forceinline__ uint32_t clusterRank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t inBlock(uint32_t address, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
    return r;
}
__device__ __forceinline__ void clusterArriveBarrier(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void clusterSync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The issuing warps run their loops as a whole, with branches that are the same for all lanes, so that descriptors and addresses live in uniform
// registers; only the elected lane's instruction (`lead`) takes effect. (Behind a `lane == 0` branch every operand is moved to a
// uniform register first: four products and a commit took 500 clocks to issue, whatever their size.)
__device__ __forceinline__ uint32_t electOne()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
template <int CTAS>
__device__ __forceinline__ void tmaLoad2(uint32_t lead, uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    // (.cta_group::2: the barrier may be the other block's; the destination is this block's own, nothing is multicast)
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n\t}"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmaLoad3(uint32_t lead, uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
                     "@q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
                     "@q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];\n\t}"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void fenceProxyAsync() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int CTAS>
__device__ __forceinline__ void mma(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t accumulate)
{
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(accumulate), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(accumulate), "r"(lead) : "memory");
}
// arrives on the barrier (of both blocks, at the same place) when the products issued so far are done
template <int CTAS>
__device__ __forceinline__ void mmaCommit(uint32_t lead, uint32_t bar)
{
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                     "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
                     "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
                     ::"r"(bar), "h"(static_cast<uint16_t>(3)), "r"(lead) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmemAlloc(uint32_t at, uint32_t columns)
{
    if constexpr (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(at), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmemFree(uint32_t at, uint32_t columns)
{
    if constexpr (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns) : "memory");
}
// 32 consecutive fp32 columns of this thread's lane of tensor memory; there after tmemWait
__device__ __forceinline__ void tmemLoad32(uint32_t at, float (&v)[32])
{
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
                   "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                   "=r"(r[30]), "=r"(r[31])
                 : "r"(at) : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// (the values are operands: nothing that uses them may move in front of the wait)
__device__ __forceinline__ void tmemWait(float (&v)[32], float (&w)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]), "+f"(w[i]));
}
// descriptor of a 128-byte swizzled operand: groups of 8 rows of 128 bytes lie 1024 bytes apart. K-major: the rows are rows of the
// operand. MN-major: the rows run along the sum, and blocks of 64 rows of the operand lie `lead` bytes apart.
__device__ __forceinline__ uint64_t operandDescriptor(uint32_t address, uint32_t lead)
{
    return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// ---- plan ------------------------------------------------------------------------------------------------------------------
enum Product : int { FORWARD = 0, INPUT = 1, WEIGHTS = 2 };
constexpr int BM = 128, BK = 64, BOX = 64 * 128;   // rows of D per block, step along the sum, bytes of a box of 64 x 64 elements
constexpr int EPILOGUE_GROUPS = 2, EPILOGUE_WARPS = 4 * EPILOGUE_GROUPS, SUM_WARPS = 4;
constexpr int EPILOGUE_BYTES = 32 * 64 + 128;      // per warp: 32 rows x 32 elements of 16 bits, 32 floats of bias
// producer, products, epilogue; the weight gradient with a bias gradient: warps that sum the columns of dy
__host__ __device__ constexpr int blockThreads(bool sums) { return (2 + EPILOGUE_WARPS + (sums ? SUM_WARPS : 0)) * 32; }

// Lists in shared memory: bounds, before, and for up to SORTED_MAX experts their order, with room to sort them in
constexpr int SORTED_MAX = 512;
__host__ __device__ constexpr int listStride(int experts) { return (experts + 4) / 4 * 4; }
__host__ __device__ constexpr int listInts(int experts) { return experts <= SORTED_MAX ? 2 * listStride(experts) + SORTED_MAX : 2 * listStride(experts); }

struct ProductArgs {
    long long rows;
    int experts, columns, sum;    // columns of D; length of the sum (forward, input), channels out (weights)
    int rowTiles, columnTiles;    // weights: tiles of D; else columnTiles alone
    int chunk;                    // weights: rows of an expert per item
    int tileRows;                 // rows of D per tile: BM x CTAS
    const int* offsets;
    void* out;
    long long outStride;          // elements between rows of D in memory
    const void* bias;             // forward: (experts, columns) or null
    const float* powers;          // input: what the sums of an expert's rows are multiplied with, or null
    int2* plan;                   // weights: first slot and items of an expert, written for the join; null where no expert can have two
    float* partial;               // weights: slots x tiles x tileRows x BN sums; the items of experts with more than one have a slot each
    int* status;
    void* gradBias;               // weights: (experts, channels out) or null
    float* partialBias;           // weights: slots x channels out sums
    bool wideStore;               // rows of D can be written 16 bytes at a time
};

// Offsets are taken as the running maximum of what they say, within [0, rows]: runs are disjoint whatever the caller's array holds.
// Without offsets every row belongs to the one expert there is.
__device__ __forceinline__ int clampOffset(const ProductArgs& p, int e)
{
    if (p.offsets == nullptr) return e == 0 ? 0 : static_cast<int>(p.rows);
    return static_cast<int>(max(0ll, min(p.rows, static_cast<long long>(p.offsets[e]))));
}
// pieces of at most `piece` rows that `rows` rows fill, and the end of one that begins at `begin` (a sum of rows and a piece can pass 31 bits)
__host__ __device__ constexpr int piecesOf(int rows, int piece) { return rows > 0 ? (rows - 1) / piece + 1 : 0; }
__host__ __device__ constexpr int pieceEnd(int begin, int piece, int last) { return last - begin > piece ? begin + piece : last; }
constexpr int MOST_ROWS = 0x7fffffff - 4095;   // what the entry points let pass
static_assert(piecesOf(MOST_ROWS, 1 << 16) == 1 << 15 && piecesOf(MOST_ROWS, 1 << 30) == 2 && piecesOf(1, 128) == 1 && piecesOf(128, 128) == 1 && piecesOf(0, 128) == 0, "");
static_assert(pieceEnd(MOST_ROWS - 10, 1 << 16, MOST_ROWS) == MOST_ROWS && pieceEnd(5, 128, 300) == 133 && pieceEnd(172, 128, 300) == 300 && pieceEnd(173, 128, 300) == 300, "");
// units of work along `rows` rows of an expert
template <int MODE>
__device__ __forceinline__ int unitsOf(const ProductArgs& p, int rows)
{
    return piecesOf(rows, MODE == WEIGHTS ? p.chunk : p.tileRows);
}
// The experts' runs and units of work, for all threads of a block: bounds[e] = first row of expert e, bounds[experts] the end of the last one;
// before[i] = units of the experts in front of the i-th in `order`. The weight product takes the longest runs first (up to SORTED_MAX
// experts): its tiles cost what their runs are long, and the blocks' shares come out even. (Segments
// of 32 experts side by side: one warp that took them one after the other cost a kernel of 512 experts 8 us.)
template <int MODE>
__device__ __forceinline__ void planExperts(const ProductArgs& p, int* bounds, int* before, int* order, int threads)
{
    __shared__ int segment[64];   // of 32 experts: their largest offset, then their units
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = threads / 32, segments = (p.experts + 31) / 32;
    const int start = clampOffset(p, 0);
    for (int s = warp; s < segments; s += warps) {   // running maximum
        const int e = s * 32 + lane;
        int end = e < p.experts ? max(start, clampOffset(p, e + 1)) : start;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, up);
        }
        if (e < p.experts) bounds[e + 1] = end;
        if (lane == 31) segment[s] = end;
    }
    if (threadIdx.x == 0) bounds[0] = start;
    __syncthreads();
    for (int s = warp; s < segments; s += warps) {
        const int e = s * 32 + lane;
        const int reached = __reduce_max_sync(0xffffffffu, max(lane < s ? segment[lane] : 0, lane + 32 < s ? segment[lane + 32] : 0));
        if (e < p.experts) bounds[e + 1] = max(bounds[e + 1], reached);
    }
    __syncthreads();
    const bool sorted = MODE == WEIGHTS && order != nullptr;
    if (sorted) {
        // bitonic, of keys (length, number) that differ, the length cut to 22 bits
        const int size = p.experts <= 1 ? 1 : 1 << (32 - __clz(p.experts - 1)), cut = max(0, 10 - __clzll(p.rows) + 32);
        unsigned* keys = reinterpret_cast<unsigned*>(before);   // (has room for SORTED_MAX, and is not needed yet)
        for (int e = threadIdx.x; e < size; e += threads) keys[e] = e < p.experts ? static_cast<unsigned>((bounds[e + 1] - bounds[e]) >> cut) << 10 | (e + 1) : 0u;
        for (int length = 2; length <= size; length *= 2)
            for (int apart = length / 2; apart > 0; apart /= 2) {
                __syncthreads();
                const int i = (threadIdx.x / apart * 2) * apart + threadIdx.x % apart;
                if (threadIdx.x < size / 2) {
                    const unsigned x = keys[i], y = keys[i + apart];
                    if ((x < y) == ((i & length) == 0)) {
                        keys[i] = y;
                        keys[i + apart] = x;
                    }
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < p.experts; i += threads) order[i] = static_cast<int>(keys[i] & 1023) - 1;
        __syncthreads();
    }
    for (int s = warp; s < segments; s += warps) {
        const int i = s * 32 + lane, e = i < p.experts ? (sorted ? order[i] : i) : 0;
        int units = i < p.experts ? unitsOf<MODE>(p, bounds[e + 1] - bounds[e]) : 0;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, units, o);
            if (lane >= o) units += up;
        }
        if (i < p.experts) before[i + 1] = units;
        if (lane == 31) segment[s] = units;
    }
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
    for (int s = warp; s < segments; s += warps) {
        const int i = s * 32 + lane;
        const int carry = __reduce_add_sync(0xffffffffu, (lane < s ? segment[lane] : 0) + (lane + 32 < s ? segment[lane + 32] : 0));
        if (i < p.experts) before[i + 1] += carry;
    }
    // (the caller's barrier follows)
}

// One tile of D: its expert (-1: no tile), the slot of its partial sums if the expert has several units, the expert's units, the run of rows it reads (forward, input: its own rows)
// and where it lies.
struct Tile {
    int expert, slot, units, begin, end, row, column;
};
// Walks the tiles of a block or pair of blocks: one of every round, from alternating ends, so that with the longest first the shares come out
// even; rounds `round`, `round` + `stride`, ... All threads of a warp call next() together: 32 experts are looked at in one step.
template <int MODE, int BN, int CTAS>
struct Walk {
    const ProductArgs* args;
    const int *bounds, *before, *order;   // planExperts
    long long total;
    int perUnit, round, stride, at = 0, singles = 0;   // at: place in `order` (the expert itself without one); singles: experts of one unit in front of it
    __device__ __forceinline__ Walk(const ProductArgs& p, const int* rows, const int* units, const int* list, int first, int step)
        : args(&p), bounds(rows), before(units), order(MODE == WEIGHTS ? list : nullptr), round(first), stride(step)
    {
        perUnit = MODE == WEIGHTS ? p.rowTiles * p.columnTiles : p.columnTiles;
        total = static_cast<long long>(before[p.experts]) * perUnit;
    }
    __device__ __forceinline__ bool next(Tile& t)
    {
        const ProductArgs& p = *args;
        const int blocks = gridDim.x / CTAS, block = blockIdx.x / CTAS;
        const long long tile = static_cast<long long>(round) * blocks + (round & 1 ? blocks - 1 - block : block);
        if (static_cast<long long>(round) * blocks >= total) return false;
        round += stride;
        t.expert = -1;
        if (tile >= total) return true;   // (the last round may have no tile for this block)
        const int unit = perUnit == 1          ? static_cast<int>(tile)
                         : total <= 0x7fffffff ? static_cast<int>(static_cast<unsigned>(tile) / static_cast<unsigned>(perUnit))
                                               : static_cast<int>(tile / perUnit);
        const int within = static_cast<int>(tile - static_cast<long long>(unit) * perUnit);
        const int lane = threadIdx.x & 31;
        for (;;) {   // first expert whose units reach behind `unit`
            const int i = at + 1 + lane;
            const bool behind = i <= p.experts && before[i] <= unit;
            const unsigned passed = __ballot_sync(0xffffffffu, behind);
            if constexpr (MODE == WEIGHTS) singles += __popc(__ballot_sync(0xffffffffu, behind && before[i] - before[i - 1] == 1));
            at += __popc(passed);
            if (passed != 0xffffffffu) break;
        }
        t.expert = order != nullptr ? order[at] : at;
        const int first = bounds[t.expert], last = bounds[t.expert + 1];
        t.slot = unit - singles;
        t.units = before[at + 1] - before[at];
        const int part = unit - before[at];
        if constexpr (MODE == WEIGHTS) {
            const int row = within / p.columnTiles;
            t.begin = first + part * p.chunk;
            t.end = pieceEnd(t.begin, p.chunk, last);
            t.row = row * (BM * CTAS);
            t.column = (within - row * p.columnTiles) * BN;
        } else {
            t.begin = first + part * (BM * CTAS);
            t.end = pieceEnd(t.begin, BM * CTAS, last);
            t.row = t.begin;
            t.column = within * BN;
        }
        return true;
    }
    // steps along the sum
    __device__ __forceinline__ int steps(const Tile& t) const { return t.expert < 0 ? 0 : MODE == WEIGHTS ? (t.end - t.begin + BK - 1) / BK : (args->sum + BK - 1) / BK; }
};

// A wait that ends, for a whole warp: on success, when another warp of the block has given up, or after WAIT_LIMIT polls. False: leave.
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, volatile int* failed)
{
    bool ok = false;
    for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
        ok = barrierTest(bar, parity);
        if (ok || ((i & 63) == 63 && *failed != 0)) break;
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) *failed = 1;
    return ok;
}

// Where the warp that issues copies has stopped. When a warp of the block has given up, whichever it was, the copies that are still on their way
// land (or are waited for to the limit) before the block's shared memory is given back.
struct InFlight {
    uint32_t stage = 0, phase = 0, tailPhase = 0, tail = 0;
    int count = 0;
    __device__ __forceinline__ void land(uint32_t full, uint32_t stages)
    {
        for (; count > 0; --count) {
            if (stage == 0) { stage = stages; phase ^= 1; }
            --stage;
            barrierWait(full + stage * 8, phase);
        }
    }
};

// A warp writes 32 rows x 32 columns of fp32 (a row per lane) from column c0 on to the rows of `out` (which has `columns` columns and `rows` rows from
// the first lane's on), through 2 KB of shared memory: rows of 64 bytes, their 16-byte chunks exchanged so that neither side meets a bank twice.
template <class T>
__device__ __forceinline__ void storeTile(const float (&v)[32], unsigned char* mine, T* out, long long stride, int rows, int c0, int columns, bool wideStore)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        store<T, 8>(reinterpret_cast<T*>(mine + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)), pack<T, 8>(*reinterpret_cast<const float (*)[8]>(&v[i * 8])));
    __syncwarp();
    if (wideStore) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 2), chunk = lane & 3, column = c0 + chunk * 8;
            if (r < rows && column < columns) store<T, 8>(out + r * stride + column, load<T, 8>(reinterpret_cast<const T*>(mine + r * 64 + ((chunk ^ ((r >> 1) & 3)) << 4))));
        }
    } else {
        const int column = c0 + lane;
        for (int r = 0; r < 32 && r < rows; ++r)
            if (column < columns) out[r * stride + column] = *reinterpret_cast<const T*>(mine + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
    }
    __syncwarp();
}

// boxes of 64 that `n` elements fill, 0 to `most`
__device__ __forceinline__ int boxes(int n, int most) { return max(0, min(most, (n + 63) / 64)); }

// ---- host ------------------------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeFn encoder()
{
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

} // namespace products
} // namespace kernel
} // namespace qmlp
