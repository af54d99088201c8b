// Matrix products grouped by expert: rows [offsets[e], offsets[e + 1]) of x belong to expert e.
//
//   forward          y_r  = W_e x_r + b_e                    W_e: (channels out, channels in)
//   input gradient   dx_r = W_e^T dy_r
//   weight gradient  dW_e = sum over the expert's rows of dy_r x_r^T        db_e = sum of dy_r
//
// One tcgen05 kernel computes all three products, D (128 x BN, fp32 in tensor memory) += A B over blocks of 64 along the sum:
//              rows of D          columns of D      sum              A                      B
//   forward    rows of x          channels out      channels in      x, K-major             W_e, K-major
//   input      rows of dy         channels in       channels out     dy, K-major            W_e read along its rows (MN-major)
//   weights    channels out       channels in       expert's rows    dy read along (MN)     x read along (MN)
// so nothing is transposed in memory. Operands arrive by TMA in boxes of 64 x 64 elements, 128-byte swizzled; what lies outside a
// matrix arrives as zeros. A tile of rows that reaches behind its expert's last row reads rows of the next expert: in the first two
// products those only fill rows of D that are not stored; in the third they are zeroed in shared memory before the tensor core
// reads them (a zero in one operand would not do: another expert's infinity times zero is NaN).
//
// One persistent block per SM, or a pair of blocks that share tiles of 256 x 256 (cta_group::2; each block loads half of either operand):
// a TMA warp, an MMA warp, two groups of four epilogue warps, one per accumulator, so that the products of a tile run under the
// epilogues of the two before; in the weight product four more warps add up the columns of dy for the bias gradient, from the
// stages that are in shared memory anyway. Which tile is whose follows from the offsets, which every block adds up for itself: the group
// sizes never travel to the host. 16 experts, 131072 rows, 1024 -> 1024 bfloat16: 200, 196 and 205 us for the three products, 3 us more
// with the bias gradient (1.34 to 1.40 PFLOP/s; a library product of one matrix of that size 198 us, at clocks that the power limit holds
// down; 128 x 256 tiles of single blocks 254, 239 and 346 us: their operands ask for more bytes a clock than shared memory has).
// 512 experts, 1000003 rows, 64 -> 64 half: forward 52 us, bound by memory (40 us at the copy rate).
// Waits are bounded: on a timeout the block drains, gives its tensor memory back and sets the library's status word.
#include "common.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include <cuda.h>

namespace qmlp {
namespace kernel {
namespace {

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

// BN: columns of D; CTAS: blocks that share a tile, each with BM rows of D and BN / CTAS of the columns of B
template <int BN, int CTAS>
struct Layout {
    static constexpr int BCOLS = BN / CTAS, ABYTES = BM * 128, BBYTES = BCOLS * 128, STAGE = ABYTES + BBYTES;
    static constexpr int STAGES = 192 * 1024 / STAGE;
    static constexpr int TMEM = 2 * BN;
    static constexpr int OUT = EPILOGUE_WARPS * EPILOGUE_BYTES;
    // barriers: full, empty, landed (STAGES each, at most 8), accumulator full, empty (2 each), tail, drain; then flag and tensor memory
    static constexpr int FULL = 0, EMPTY = 64, LANDED = 128, ACC_FULL = 192, ACC_EMPTY = 208, TAIL = 224, DRAIN = 232, FAILED = 240, BASE = 244, BARS = 256;
    // 1 KB for the alignment of the ring
    static constexpr int bytes(int experts) { return 1024 + STAGES * STAGE + OUT + BARS + listInts(experts) * 4; }
    static_assert(STAGES <= 8, "barriers");
    static_assert(bytes(EXPERTS_MAX) + 512 <= 227 * 1024, "shared memory");
};

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
    int2* plan;                   // weights: first slot and items of an expert, written for the join; null where no expert can have two
    float* partial;               // weights: slots x tiles x tileRows x BN sums; the items of experts with more than one have a slot each
    int* status;
    void* gradBias;               // weights: (experts, channels out) or null
    float* partialBias;           // weights: slots x channels out sums
    bool wideStore;               // rows of D can be written 16 bytes at a time
};

// Offsets are taken as the running maximum of what they say, within [0, rows]: runs are disjoint whatever the caller's array holds.
__device__ __forceinline__ int clampOffset(const ProductArgs& p, int e)
{
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

// barrier over the four warps that sum, with the conjunction of their answers
__device__ __forceinline__ bool sumWarpsAgree(bool answer)
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(static_cast<uint32_t>(answer)) : "memory");
    return r != 0;
}

// operand format in the instruction descriptor
template <class T> constexpr uint32_t FORMAT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;

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

// `n` zeros, by a warp
constexpr int ZERO_PIECE = 4096;
template <class T>
__device__ __forceinline__ void zeroRun(T* at, int n)
{
    const int lane = threadIdx.x & 31, head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) / 2), wide = (n - head) / 8, tail = head + wide * 8;
    if (lane < head) at[lane] = Element<T>::from(0.f);
    for (int i = lane; i < wide; i += 32) store<T, 8>(at + head + i * 8, Pack<T, 8>{});
    if (tail + lane < n) at[tail + lane] = Element<T>::from(0.f);
}

// boxes of 64 that `n` elements fill, 0 to `most`
__device__ __forceinline__ int boxes(int n, int most) { return max(0, min(most, (n + 63) / 64)); }

template <class T, int MODE, int BN, int CTAS, bool SUMS>
__global__ void __launch_bounds__(blockThreads(SUMS), 1)
    expert_product_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ ProductArgs p)
{
    using L = Layout<BN, CTAS>;
    extern __shared__ unsigned char dynamic[];
    const uint32_t raw = smemAddress(dynamic), ring = (raw + 1023u) & ~1023u;
    unsigned char* base = dynamic + (ring - raw);
    unsigned char* outStage = base + L::STAGES * L::STAGE;
    const uint32_t bars = ring + L::STAGES * L::STAGE + L::OUT;
    const uint32_t full = bars + L::FULL, empty = bars + L::EMPTY, landed = bars + L::LANDED, accFull = bars + L::ACC_FULL, accEmpty = bars + L::ACC_EMPTY;
    volatile int* failed = reinterpret_cast<volatile int*>(outStage + L::OUT + L::FAILED);
    uint32_t* tmemBase = reinterpret_cast<uint32_t*>(outStage + L::OUT + L::BASE);
    int *bounds = reinterpret_cast<int*>(outStage + L::OUT + L::BARS), *before = bounds + listStride(p.experts);
    int* order = p.experts <= SORTED_MAX ? before + listStride(p.experts) : nullptr;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 1 ? 0u : clusterRank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            barrierInit(full + s * 8, CTAS);
            barrierInit(empty + s * 8, 1);
            barrierInit(landed + s * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrierInit(accFull + i * 8, 1);
            barrierInit(accEmpty + i * 8, 4 * CTAS);
        }
        barrierInit(bars + L::TAIL, 1);
        barrierInit(bars + L::DRAIN, 1);
        *failed = 0;
        barrierInitDone();
    }
    if (warp == 1) tmemAlloc<CTAS>(smemAddress(tmemBase), L::TMEM);
    chained();
    planExperts<MODE>(p, bounds, before, order, blockThreads(SUMS));
    fenceBefore();
    __syncthreads();
    if constexpr (CTAS > 1) clusterSync();   // the other block's barriers are set
    fenceAfter();
    const uint32_t tmem = *tmemBase;
    Walk<MODE, BN, CTAS> walk(p, bounds, before, order, 0, 1);
    Tile t;
    InFlight copies;   // of warp 0

    if (warp == 0) {
        // ---- operands -------------------------------------------------------------------------------------------------
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0, tailPhase = 0;
        long long issued = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            const int steps = walk.steps(t);
            const int row = t.row + rank * BM, column = t.column + rank * L::BCOLS, rowEnd = MODE == WEIGHTS ? p.sum : t.end;
            const int boxesA = boxes(rowEnd - row, BM / 64), boxesB = boxes(p.columns - column, L::BCOLS / 64);
            const uint32_t bytes = (boxesA + boxesB) * BOX;   // of this block; of both blocks:
            const uint32_t allBytes = CTAS == 1 ? bytes : bytes + (boxes(rowEnd - row - BM, BM / 64) + boxes(p.columns - column - L::BCOLS, L::BCOLS / 64)) * BOX;
            for (int k = 0; __all_sync(0xffffffffu, k < steps); ++k) {
                if (!await(empty + stage * 8, phase ^ 1, failed)) { ok = false; break; }
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES;
                const uint32_t ready = CTAS == 1 ? full + stage * 8 : inBlock(full + stage * 8, 0);
                // the last rows of an expert's last step belong to another expert: a pair of blocks clears them before it hands the step on
                const int left = t.end - t.begin - k * BK, tail = MODE == WEIGHTS && CTAS > 1 && left < BK ? (16 - left % 16) % 16 : 0;
                const uint32_t bar = tail > 0 ? bars + L::TAIL : ready;
                if (lead) {
                    // the leader expects the bytes of both blocks, and arrives for both (an arrival from the other block at every step costs more
                    // than the step: its release takes about a microsecond)
                    if (tail > 0) barrierExpect(bar, bytes);
                    else if (rank == 0) {
                        barrierExpect(full + stage * 8, allBytes);
                        if (CTAS > 1) barrierArrive(full + stage * 8);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < BM / 64; ++i) {
                    if constexpr (MODE == WEIGHTS) tmaLoad2<CTAS>(lead && i < boxesA, a + i * BOX, &mapA, row + i * 64, t.begin + k * BK, bar);
                    else tmaLoad2<CTAS>(lead && i < boxesA, a + i * BOX, &mapA, k * BK, row + i * 64, bar);
                }
#pragma unroll
                for (int i = 0; i < L::BCOLS / 64; ++i) {
                    if constexpr (MODE == WEIGHTS) tmaLoad2<CTAS>(lead && i < boxesB, b + i * BOX, &mapB, column + i * 64, t.begin + k * BK, bar);
                    else if constexpr (MODE == FORWARD) tmaLoad3<CTAS>(lead && i < boxesB, b + i * BOX, &mapB, k * BK, column + i * 64, t.expert, bar);
                    else tmaLoad3<CTAS>(lead && i < boxesB, b + i * BOX, &mapB, column + i * 64, k * BK, t.expert, bar);
                }
                if constexpr (MODE == WEIGHTS && CTAS > 1) {
                    if (tail > 0) {
                        if (!await(bar, tailPhase, failed)) { copies.tail = 1; ok = false; break; }
                        tailPhase ^= 1;
                        for (int i = lane; i < tail * (L::STAGE / BOX) * 8; i += 32) {
                            const int box = i / (tail * 8), r = left + i / 8 % tail, chunk = i % 8;
                            *reinterpret_cast<uint4*>(base + stage * L::STAGE + box * BOX + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fenceProxyAsync();
                        __syncwarp();
                        if (lane == 0) clusterArriveBarrier(ready);
                        __syncwarp();
                    }
                }
                ++issued;
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        copies.stage = stage;
        copies.phase = phase;
        copies.tailPhase = tailPhase;
        copies.count = rank == 0 ? static_cast<int>(min(issued, static_cast<long long>(L::STAGES))) : 0;   // (the other block's arrive here too)
    } else if (warp == 1) {
        // ---- products -------------------------------------------------------------------------------------------------
        constexpr uint32_t instruction = (1u << 4) | (FORMAT<T> << 7) | (FORMAT<T> << 10) | (MODE == WEIGHTS ? 1u << 15 : 0u) | (MODE != FORWARD ? 1u << 16 : 0u) |
                                         (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>((BM * CTAS) >> 4) << 24);
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0, acc = 1, accPhases = 0;   // accPhases: one bit per accumulator
        bool ok = rank == 0;
        while (ok && walk.next(t)) {
            const int steps = walk.steps(t);
            acc ^= 1;                   // the tiles' numbers alternate between the accumulators
            if (__all_sync(0xffffffffu, steps == 0)) continue;   // no tile for this block in the last round
            if (!await(accEmpty + acc * 8, (accPhases >> acc & 1) ^ 1, failed)) break;
            accPhases ^= 1u << acc;
            fenceAfter();
            const uint32_t d = tmem + acc * BN;
            for (int k = 0; __all_sync(0xffffffffu, k < steps); ++k) {
                if (!await(full + stage * 8, phase, failed)) { ok = false; break; }
                fenceAfter();
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES;
                const int left = MODE == WEIGHTS ? t.end - t.begin - k * BK : p.sum - k * BK, parts = min(BK, left + 15) / 16;
                if (MODE == WEIGHTS && CTAS == 1 && left < parts * 16) {
                    // the last rows of the step belong to another expert
                    const int rows = parts * 16 - left;
                    for (int i = lane; i < rows * (L::STAGE / BOX) * 8; i += 32) {
                        const int box = i / (rows * 8), r = left + i / 8 % rows, chunk = i % 8;
                        *reinterpret_cast<uint4*>(base + stage * L::STAGE + box * BOX + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fenceProxyAsync();
                    __syncwarp();
                }
                const uint64_t descA = operandDescriptor(a, MODE == WEIGHTS ? BOX : 16), descB = operandDescriptor(b, MODE == FORWARD ? 16 : BOX);
                // 16 along the sum: 32 bytes of a K-major row, 16 rows of an MN-major block
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma<CTAS>(lead && i < parts, d, descA + i * (MODE == WEIGHTS ? 2048 >> 4 : 32 >> 4), descB + i * (MODE == FORWARD ? 32 >> 4 : 2048 >> 4), instruction,
                              i > 0 ? 1u : k > 0 ? 1u : 0u);
                mmaCommit<CTAS>(lead, (SUMS && t.column == 0 ? landed : empty) + stage * 8);   // (the warps that sum come between)
                mmaCommit<CTAS>(lead && k == steps - 1, accFull + acc * 8);
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp < 2 + EPILOGUE_WARPS) {
        // ---- epilogue: two groups of four warps, one per accumulator -------------------------------------------------------
        const int group = (warp - 2) / 4, quarter = warp & 3;   // quarter: lanes of tensor memory this warp may read
        unsigned char* mine = outStage + (warp - 2) * EPILOGUE_BYTES;
        float* mineBias = reinterpret_cast<float*>(mine + 32 * 64);
        const uint32_t released = CTAS == 1 ? accEmpty + group * 8 : inBlock(accEmpty + group * 8, 0);
        T* out = static_cast<T*>(p.out);
        uint32_t accPhase = 0;
        if (MODE == WEIGHTS && p.plan != nullptr && blockIdx.x == 0 && warp == 2) {   // for the kernel that joins the partial sums
            int singles = 0;
            for (int i = lane; i - lane < p.experts; i += 32) {
                const int units = i < p.experts ? before[i + 1] - before[i] : 0;
                const unsigned single = __ballot_sync(0xffffffffu, units == 1);
                if (i < p.experts) p.plan[order != nullptr ? order[i] : i] = make_int2(before[i] - singles - __popc(single & ((1u << lane) - 1)), units);
                singles += __popc(single);
            }
        }
        if constexpr (MODE == WEIGHTS) {
            // the gradients of experts without rows, while the first products run (as tiles without products: 431 experts of 66 -> 760, 19 rows, 40 us;
            // so 22 us)
            const long long matrix = static_cast<long long>(p.sum) * p.columns;
            const int pieces = static_cast<int>((matrix + ZERO_PIECE - 1) / ZERO_PIECE), warps = gridDim.x * EPILOGUE_WARPS;
            for (long long i = blockIdx.x * EPILOGUE_WARPS + (warp - 2); i < static_cast<long long>(p.experts) * pieces; i += warps) {
                const int e = static_cast<int>(i / pieces), piece = static_cast<int>(i - static_cast<long long>(e) * pieces);
                if (bounds[e + 1] > bounds[e]) continue;
                const long long first = static_cast<long long>(piece) * ZERO_PIECE;
                zeroRun<T>(out + e * matrix + first, static_cast<int>(min(static_cast<long long>(ZERO_PIECE), matrix - first)));
                if (SUMS && piece == 0) zeroRun<T>(static_cast<T*>(p.gradBias) + static_cast<long long>(e) * p.sum, p.sum);
            }
        }
        walk = Walk<MODE, BN, CTAS>(p, bounds, before, order, group, EPILOGUE_GROUPS);
        while (walk.next(t)) {
            if (t.expert < 0) break;
            const int tileRow = t.row + rank * BM;
            float bias[BN / 32];   // of column c * 32 + lane
            if constexpr (MODE == FORWARD) {
                const T* row = static_cast<const T*>(p.bias) + static_cast<long long>(t.expert) * p.columns + t.column;
#pragma unroll
                for (int i = 0; i < BN / 32; ++i) bias[i] = p.bias != nullptr && t.column + i * 32 + lane < p.columns ? Element<T>::to(row[i * 32 + lane]) : 0.f;
            }
            if (!await(accFull + group * 8, accPhase, failed)) break;
            accPhase ^= 1;
            fenceAfter();
            const uint32_t from = tmem + group * BN + (static_cast<uint32_t>(quarter * 32) << 16);
            // rows of D in memory: expert by expert, channels out (weights); the tile's own rows (else)
            const int rowsLeft = (MODE == WEIGHTS ? p.sum : t.end) - tileRow - quarter * 32;
            const long long firstRow = (MODE == WEIGHTS ? static_cast<long long>(t.expert) * p.sum : 0ll) + tileRow + quarter * 32;
            const bool split = MODE == WEIGHTS && t.units > 1;
            float* partial = nullptr;
            if constexpr (MODE == WEIGHTS) {
                const long long slot = t.slot, tileAt = static_cast<long long>(t.row / (BM * CTAS)) * p.columnTiles + t.column / BN;
                partial = p.partial + ((slot * p.rowTiles * p.columnTiles + tileAt) * (BM * CTAS) + rank * BM + quarter * 32 + lane) * BN;
            }
            // 64 columns of the accumulator at a time, 32 through shared memory
#pragma unroll
            for (int pair = 0; pair < BN / 64; ++pair) {
                if (t.column + pair * 64 >= p.columns || rowsLeft <= 0) break;
                float v[2][32];
                tmemLoad32(from + pair * 64, v[0]);
                tmemLoad32(from + pair * 64 + 32, v[1]);
                tmemWait(v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c0 = pair * 64 + h * 32;
                    if (t.column + c0 >= p.columns) break;
                    if (split) {
                        if (lane < rowsLeft) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(partial + c0 + i) = make_float4(v[h][i], v[h][i + 1], v[h][i + 2], v[h][i + 3]);
                        }
                        __syncwarp();   // (the next load of tensor memory is the whole warp's)
                        continue;
                    }
                    if constexpr (MODE == FORWARD) {
                        if (p.bias != nullptr) {
                            mineBias[lane] = bias[pair * 2 + h];
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 f = *reinterpret_cast<const float4*>(mineBias + i);
                                v[h][i] += f.x;
                                v[h][i + 1] += f.y;
                                v[h][i + 2] += f.z;
                                v[h][i + 3] += f.w;
                            }
                        }
                    }
                    storeTile<T>(v[h], mine, out + firstRow * p.outStride + t.column, p.outStride, rowsLeft, c0, p.columns - t.column, p.wideStore);
                }
            }
            fenceBefore();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CTAS == 1) barrierArrive(released);
                else clusterArriveBarrier(released);
            }
        }
        if constexpr (MODE != WEIGHTS) {
            // rows before the first and behind the last expert belong to nobody
            const int first = bounds[0], last = bounds[p.experts];
            const long long threads = static_cast<long long>(gridDim.x) * EPILOGUE_WARPS, me = static_cast<long long>(blockIdx.x) * EPILOGUE_WARPS + (warp - 2);
            for (long long r = me; r < first + (p.rows - last); r += threads) {
                T* row = out + (r < first ? r : last + (r - first)) * p.outStride;
                for (int c = lane; c < p.columns; c += 32) row[c] = Element<T>::from(0.f);
            }
        }
    } else if constexpr (SUMS) {
        // ---- bias gradient: the columns of dy, summed where they lie for the products ----------------------------------------
        // A thread takes 8 columns (a 16-byte chunk) of every eighth row of a step, when the products of the step are done and before its
        // stage is handed back; only tiles of the first columns count.
        const int thread = threadIdx.x - (2 + EPILOGUE_WARPS) * 32;
        const int chunk = thread >> 3, first = thread & 7;   // chunk of the 16 chunks of 128 columns; 8 neighbouring lanes share one
        uint32_t stage = 0, phases = 0;                      // phases: one bit per stage
        bool ok = true;
        while (ok && walk.next(t)) {
            const int steps = walk.steps(t);
            if (t.expert < 0) break;
            if (t.column != 0) {
                stage = (stage + steps) % L::STAGES;
                continue;
            }
            const int tileRow = t.row + rank * BM;
            float2 sum[4] = {};
            for (int k = 0; k < steps; ++k) {
                // (the four warps leave together: none may wait for another below)
                if (!sumWarpsAgree(await(landed + stage * 8, phases >> stage & 1, failed))) { ok = false; break; }
                phases ^= 1u << stage;
                const int left = t.end - t.begin - k * BK;
                const unsigned char* box = base + stage * L::STAGE + (chunk >> 3) * BOX;
                Pack<T, 8> v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = i * 8 + first;
                    v[i] = load<T, 8>(reinterpret_cast<const T*>(box + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)));
                }
                if (left < BK) {   // rows of another expert
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i * 8 + first >= left) v[i] = {};
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum[j] = add2(sum[j], toPair(&v[i].v[2 * j]));
                __syncwarp();
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (thread == 0) barrierArrive(empty + stage * 8);
                if (++stage == L::STAGES) stage = 0;
            }
            if (ok) {
                float mine = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float all = groupSum<8>(j % 2 == 0 ? sum[j / 2].x : sum[j / 2].y);
                    mine = first == j ? all : mine;
                }
                const int channel = tileRow + chunk * 8 + first;
                if (channel < p.sum) {
                    if (t.units > 1) p.partialBias[static_cast<long long>(t.slot) * p.sum + channel] = mine;
                    else static_cast<T*>(p.gradBias)[static_cast<long long>(t.expert) * p.sum + channel] = Element<T>::from(mine);
                }
            }
        }
    }
    fenceBefore();
    __syncthreads();
    fenceAfter();
    if (*failed != 0 && warp == 0) {
        copies.land(full, L::STAGES);
        if (copies.tail) barrierWait(bars + L::TAIL, copies.tailPhase);
        __syncwarp();
    }
    if (*failed != 0 && warp == 1 && rank == 0) {
        // products that were issued end before the tensor memory is given back
        mmaCommit<CTAS>(electOne(), bars + L::DRAIN);   // (elects the lane that issued the products)
        if (lane == 0) {
            barrierWait(bars + L::DRAIN, 0);
            atomicOr(p.status, 1);
        }
        __syncwarp();
    }
    if constexpr (CTAS > 1) clusterSync();   // nothing reaches the other block any more
    if (warp == 1) tmemFree<CTAS>(tmem, L::TMEM);
}

// ---- both gradients of a narrow layer in one pass --------------------------------------------------------------------------------
// Up to 128 channels in and out, the two gradients are bound by memory, and both read dy: here a tile of 128 rows of dy and x is fetched once, and
// four operands are read from it: dy K-major and the expert's matrix for the input gradient, dy and x along their rows for the weight
// gradient, whose accumulator stays in tensor memory for as long as the block's rows belong to one expert. Blocks take consecutive tiles, an equal
// share each. An expert whose tiles lie in several blocks leaves partial sums, at most two per block (the run a block begins with, if it began
// before; the run it ends with, if it goes on), which a second kernel adds up in order.
// Four warps add up dy's columns (the bias gradient) and write the weight gradients. 512 experts, 1000003 rows, 64 -> 64 half: 73 us and 7 us for
// the sums (apart: 49 us for the input gradient, 64 and 7 us for the others).
template <int NB, int KB>   // boxes of 64 channels out, channels in
struct NarrowLayout {
    static constexpr int TILE = 128 * 128;                    // 128 rows x 64 elements
    static constexpr int STAGE = (NB + KB) * TILE, MATRIX = NB * KB * BOX;
    static constexpr int STAGES = (NB + KB) == 2 ? 5 : (NB + KB) == 3 ? 3 : 2;
    static constexpr int COLUMNS = KB * 64, TMEM = 4 * COLUMNS;   // two accumulators of either gradient
    static constexpr int OUT = EPILOGUE_WARPS * 32 * 64;
    // barriers: full, empty, landed (8 each); matrix full, empty; input gradient full, empty; weight gradient full, empty (2 each); drain; flag, tensor memory
    static constexpr int FULL = 0, EMPTY = 64, LANDED = 128, W_FULL = 192, W_EMPTY = 208, DX_FULL = 224, DX_EMPTY = 240, DW_FULL = 256, DW_EMPTY = 272, DRAIN = 288,
                         FAILED = 296, BASE = 300, BARS = 320;
    static constexpr int bytes(int experts) { return 1024 + STAGES * STAGE + 2 * MATRIX + OUT + BARS + listInts(experts) * 4; }
    static_assert(bytes(EXPERTS_MAX) + 512 <= 227 * 1024, "shared memory");
};

// the tiles of a block, one after the other
struct NarrowTile {
    int expert, begin, end;   // its rows
    bool first, last;         // of the expert's tiles in this block
    bool entered, leaves;     // the expert's tiles began in an earlier block, go on in a later one
};
struct NarrowWalk {
    const int *bounds, *before;
    int tile, firstTile, end, expert = 0;
    __device__ __forceinline__ NarrowWalk(const int* rows, const int* units, int experts) : bounds(rows), before(units)
    {
        const long long total = before[experts];
        firstTile = tile = static_cast<int>(total * blockIdx.x / gridDim.x);
        end = static_cast<int>(total * (blockIdx.x + 1) / gridDim.x);
    }
    __device__ __forceinline__ bool next(NarrowTile& t, int experts)
    {
        if (tile >= end) return false;
        const int lane = threadIdx.x & 31;
        for (;;) {   // first expert whose tiles reach behind `tile`
            const int e = expert + 1 + lane;
            const unsigned passed = __ballot_sync(0xffffffffu, e <= experts && before[e] <= tile);
            expert += __popc(passed);
            if (passed != 0xffffffffu) break;
        }
        const int from = before[expert], to = before[expert + 1];
        t.expert = expert;
        t.begin = bounds[expert] + (tile - from) * BM;
        t.end = pieceEnd(t.begin, BM, bounds[expert + 1]);
        t.first = tile == from || tile == firstTile;
        t.last = tile == to - 1 || tile == end - 1;
        t.entered = from < firstTile;
        t.leaves = to > end;
        ++tile;
        return true;
    }
};

template <class T, int NB, int KB, bool SUMS>
__global__ void __launch_bounds__(blockThreads(true), 1)
    expert_narrow_adjoint_kernel(const __grid_constant__ CUtensorMap mapY, const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW,
                                 const __grid_constant__ ProductArgs p, T* __restrict__ gradX, long long gradXStride, bool wideX)
{
    // p.columns: channels in, p.sum: channels out, p.out: weight gradient
    using L = NarrowLayout<NB, KB>;
    extern __shared__ unsigned char dynamic[];
    const uint32_t raw = smemAddress(dynamic), ring = (raw + 1023u) & ~1023u;
    unsigned char* base = dynamic + (ring - raw);
    const uint32_t matrices = ring + L::STAGES * L::STAGE;
    unsigned char* outStage = base + L::STAGES * L::STAGE + 2 * L::MATRIX;
    unsigned char* control = outStage + L::OUT;
    const uint32_t bars = smemAddress(control);
    volatile int* failed = reinterpret_cast<volatile int*>(control + L::FAILED);
    uint32_t* tmemBase = reinterpret_cast<uint32_t*>(control + L::BASE);
    int *bounds = reinterpret_cast<int*>(control + L::BARS), *before = bounds + listStride(p.experts);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    constexpr int THREADS = blockThreads(true);

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            barrierInit(bars + L::FULL + s * 8, 1);
            barrierInit(bars + L::EMPTY + s * 8, SUMS ? SUM_WARPS : 1);
            barrierInit(bars + L::LANDED + s * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrierInit(bars + L::W_FULL + i * 8, 1);
            barrierInit(bars + L::W_EMPTY + i * 8, 1);
            barrierInit(bars + L::DX_FULL + i * 8, 1);
            barrierInit(bars + L::DX_EMPTY + i * 8, 4);
            barrierInit(bars + L::DW_FULL + i * 8, 1);
            barrierInit(bars + L::DW_EMPTY + i * 8, 4);
        }
        barrierInit(bars + L::DRAIN, 1);
        *failed = 0;
        barrierInitDone();
    }
    if (warp == 1) tmemAlloc<1>(smemAddress(tmemBase), L::TMEM);
    chained();
    planExperts<INPUT>(p, bounds, before, nullptr, THREADS);
    fenceBefore();
    __syncthreads();
    fenceAfter();
    const uint32_t tmem = *tmemBase, tmemW = tmem + 2 * L::COLUMNS;
    if (blockIdx.x == 0)   // for the kernel that joins the partial sums
        for (int e = threadIdx.x; e <= p.experts; e += THREADS) reinterpret_cast<int*>(p.plan)[e] = before[e];
    NarrowWalk walk(bounds, before, p.experts);
    NarrowTile t;
    InFlight copies, matricesIn;   // of warp 0

    if (warp == 0) {
        // ---- operands -------------------------------------------------------------------------------------------------
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0, matrix = 0, matrixPhase = 0;
        int issued = 0, matricesIssued = 0;
        bool ok = true;
        while (ok && walk.next(t, p.experts)) {
            if (__all_sync(0xffffffffu, t.first)) {
                if (!await(bars + L::W_EMPTY + matrix * 8, matrixPhase ^ 1, failed)) break;
                const uint32_t bar = bars + L::W_FULL + matrix * 8;
                if (lead) barrierExpect(bar, L::MATRIX);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int n = 0; n < NB; ++n) tmaLoad3<1>(lead, matrices + matrix * L::MATRIX + (k * NB + n) * BOX, &mapW, k * 64, n * 64, t.expert, bar);
                ++matricesIssued;
                if (++matrix == 2) { matrix = 0; matrixPhase ^= 1; }
            }
            if (!await(bars + L::EMPTY + stage * 8, phase ^ 1, failed)) { ok = false; break; }
            const uint32_t at = ring + stage * L::STAGE, bar = bars + L::FULL + stage * 8;
            const int halves = boxes(t.end - t.begin, 2);   // of 64 rows
            if (lead) barrierExpect(bar, halves * (NB + KB) * BOX);
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < NB; ++n) tmaLoad2<1>(lead && h < halves, at + n * L::TILE + h * BOX, &mapY, n * 64, t.begin + h * 64, bar);
#pragma unroll
                for (int k = 0; k < KB; ++k) tmaLoad2<1>(lead && h < halves, at + (NB + k) * L::TILE + h * BOX, &mapX, k * 64, t.begin + h * 64, bar);
            }
            ++issued;
            if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
        }
        copies.stage = stage;
        copies.phase = phase;
        copies.count = min(issued, L::STAGES);
        matricesIn.stage = matrix;
        matricesIn.phase = matrixPhase;
        matricesIn.count = min(matricesIssued, 2);
    } else if (warp == 1) {
        // ---- products -------------------------------------------------------------------------------------------------
        constexpr uint32_t shape = (1u << 4) | (FORMAT<T> << 7) | (FORMAT<T> << 10) | (1u << 16) | (static_cast<uint32_t>(L::COLUMNS >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
        constexpr uint32_t inputShape = shape, weightShape = shape | 1u << 15;   // the matrix, x along their rows; dy too in the weight gradient
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0, matrix = 1, matrixPhases = 0, dx = 0, dxPhase = 0, dwPhases = 0;   // `matrix`: also the weight gradient's accumulator
        bool ok = true;
        while (ok && walk.next(t, p.experts)) {
            if (__all_sync(0xffffffffu, t.first)) {
                matrix ^= 1;
                if (!await(bars + L::W_FULL + matrix * 8, matrixPhases >> matrix & 1, failed)) break;
                if (!await(bars + L::DW_EMPTY + matrix * 8, (dwPhases >> matrix & 1) ^ 1, failed)) break;
                matrixPhases ^= 1u << matrix;
                dwPhases ^= 1u << matrix;
            }
            if (!await(bars + L::FULL + stage * 8, phase, failed)) break;
            if (!await(bars + L::DX_EMPTY + dx * 8, dxPhase ^ 1, failed)) break;
            fenceAfter();
            const uint32_t y = ring + stage * L::STAGE, x = y + NB * L::TILE;
            const int rows = t.end - t.begin, parts = (rows + 15) / 16;
            if (__all_sync(0xffffffffu, rows < parts * 16)) {   // the rows behind belong to another expert
                const int clear = parts * 16 - rows;
                for (int i = lane; i < clear * (NB + KB) * 8; i += 32) {
                    const int tile = i / (clear * 8), r = rows + i / 8 % clear, chunk = i % 8;
                    *reinterpret_cast<uint4*>(base + stage * L::STAGE + tile * L::TILE + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
                }
                fenceProxyAsync();
                __syncwarp();
            }
            // input gradient: sum over the channels out
            const uint64_t w = operandDescriptor(matrices + matrix * L::MATRIX, NB * BOX);
#pragma unroll
            for (int n = 0; n < NB * 4; ++n)
                mma<1>(lead && n * 16 < p.sum, tmem + dx * L::COLUMNS, operandDescriptor(y + n / 4 * L::TILE, 16) + (n % 4) * (32 >> 4), w + n * (2048 >> 4), inputShape, n > 0);
            mmaCommit<1>(lead, bars + L::DX_FULL + dx * 8);
            // weight gradient: sum over the rows
            const uint64_t a = operandDescriptor(y, L::TILE), b = operandDescriptor(x, L::TILE);
#pragma unroll
            for (int r = 0; r < 8; ++r)
                mma<1>(lead && r < parts, tmemW + matrix * L::COLUMNS, a + r * (2048 >> 4), b + r * (2048 >> 4), weightShape, r > 0 || !t.first);
            mmaCommit<1>(lead, bars + (SUMS ? L::LANDED : L::EMPTY) + stage * 8);
            mmaCommit<1>(lead && t.last, bars + L::DW_FULL + matrix * 8);
            mmaCommit<1>(lead && t.last, bars + L::W_EMPTY + matrix * 8);
            if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            if (++dx == 2) { dx = 0; dxPhase ^= 1; }
        }
    } else if (warp < 2 + EPILOGUE_WARPS) {
        // ---- input gradient: two groups of four warps, one per accumulator ------------------------------------------------------
        const int group = (warp - 2) / 4, quarter = warp & 3;
        unsigned char* mine = outStage + (warp - 2) * 32 * 64;
        uint32_t phase = 0;
        int turn = 1;
        while (walk.next(t, p.experts)) {
            turn ^= 1;
            if (turn != group) continue;
            if (!await(bars + L::DX_FULL + group * 8, phase, failed)) break;
            phase ^= 1;
            fenceAfter();
            const uint32_t from = tmem + group * L::COLUMNS + (static_cast<uint32_t>(quarter * 32) << 16);
            const int rowsLeft = t.end - t.begin - quarter * 32;
            T* out = gradX + static_cast<long long>(t.begin + quarter * 32) * gradXStride;
#pragma unroll
            for (int pair = 0; pair < KB; ++pair) {
                if (pair * 64 >= p.columns || rowsLeft <= 0) break;
                float v[2][32];
                tmemLoad32(from + pair * 64, v[0]);
                tmemLoad32(from + pair * 64 + 32, v[1]);
                tmemWait(v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (pair * 64 + h * 32 < p.columns) storeTile<T>(v[h], mine, out, gradXStride, rowsLeft, pair * 64 + h * 32, p.columns, wideX);
            }
            fenceBefore();
            __syncwarp();
            if (lane == 0) barrierArrive(bars + L::DX_EMPTY + group * 8);
        }
        // rows before the first and behind the last expert belong to nobody
        const int first = bounds[0], last = bounds[p.experts];
        const long long threads = static_cast<long long>(gridDim.x) * EPILOGUE_WARPS, me = static_cast<long long>(blockIdx.x) * EPILOGUE_WARPS + (warp - 2);
        for (long long r = me; r < first + (p.rows - last); r += threads) {
            T* row = gradX + (r < first ? r : last + (r - first)) * gradXStride;
            for (int c = lane; c < p.columns; c += 32) row[c] = Element<T>::from(0.f);
        }
    } else {
        // ---- weight and bias gradients -----------------------------------------------------------------------------------------
        const int thread = threadIdx.x - (2 + EPILOGUE_WARPS) * 32, quarter = warp & 3;
        constexpr int CHUNKS = NB * 8, SHARES = 128 / CHUNKS;   // 16-byte chunks of a row of dy; threads that share one (8 or 16 neighbouring lanes)
        const int chunk = thread / SHARES, share = thread % SHARES;
        T *gradW = static_cast<T*>(p.out), *gradB = static_cast<T*>(p.gradBias);
        // experts without rows
        for (int e = blockIdx.x; e < p.experts; e += gridDim.x) {
            if (bounds[e + 1] > bounds[e]) continue;
            for (long long i = thread; i < static_cast<long long>(p.sum) * p.columns; i += 128) gradW[static_cast<long long>(e) * p.sum * p.columns + i] = Element<T>::from(0.f);
            if (SUMS)
                for (int i = thread; i < p.sum; i += 128) gradB[static_cast<long long>(e) * p.sum + i] = Element<T>::from(0.f);
        }
        uint32_t stage = 0, phase = 0, acc = 1, accPhases = 0;
        float2 sum[4] = {};
        bool ok = true;
        while (ok && walk.next(t, p.experts)) {
            if (t.first) acc ^= 1;
            const int rows = t.end - t.begin;
            if constexpr (SUMS) {
                if (!await(bars + L::LANDED + stage * 8, phase, failed)) break;
                const unsigned char* tile = base + stage * L::STAGE + (chunk >> 3) * L::TILE;
#pragma unroll
                for (int i0 = 0; i0 < 128 / SHARES; i0 += 8) {
                    Pack<T, 8> v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = (i0 + i) * SHARES + share;
                        v[i] = load<T, 8>(reinterpret_cast<const T*>(tile + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)));
                        if (r >= rows) v[i] = {};   // rows of another expert
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[j] = add2(sum[j], toPair(&v[i].v[2 * j]));
                }
                __syncwarp();
                if (lane == 0) barrierArrive(bars + L::EMPTY + stage * 8);
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
            if (!t.last) continue;
            // the block's last tile of this expert
            const bool whole = !t.entered && !t.leaves;
            const long long slot = static_cast<long long>(blockIdx.x) * 2 + (t.entered ? 0 : 1);
            if constexpr (SUMS) {
                float mine = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float all = groupSum<SHARES>(j % 2 == 0 ? sum[j / 2].x : sum[j / 2].y);
                    mine = share == j ? all : mine;
                }
                const int channel = chunk * 8 + share;
                if (share < 8 && channel < p.sum) {
                    if (whole) gradB[static_cast<long long>(t.expert) * p.sum + channel] = Element<T>::from(mine);
                    else p.partialBias[slot * 128 + channel] = mine;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = make_float2(0.f, 0.f);
            }
            if (!await(bars + L::DW_FULL + acc * 8, accPhases >> acc & 1, failed)) break;
            accPhases ^= 1u << acc;
            fenceAfter();
            const uint32_t from = tmemW + acc * L::COLUMNS + (static_cast<uint32_t>(quarter * 32) << 16);
            const int n = quarter * 32 + lane;   // this lane's channel out
#pragma unroll
            for (int pair = 0; pair < KB; ++pair) {
                float v[2][32];
                tmemLoad32(from + pair * 64, v[0]);
                tmemLoad32(from + pair * 64 + 32, v[1]);
                tmemWait(v[0], v[1]);
                if (n < p.sum) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c0 = pair * 64 + h * 32;
                        if (!whole) {
                            float* to = p.partial + (slot * 128 + n) * L::COLUMNS + c0;
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(v[h][i], v[h][i + 1], v[h][i + 2], v[h][i + 3]);
                        } else {
                            T* to = gradW + (static_cast<long long>(t.expert) * p.sum + n) * p.columns + c0;
                            if (p.wideStore) {
#pragma unroll
                                for (int i = 0; i < 32; i += 8)
                                    if (c0 + i < p.columns) store<T, 8>(to + i, pack<T, 8>(*reinterpret_cast<const float (*)[8]>(&v[h][i])));
                            } else {
#pragma unroll
                                for (int i = 0; i < 32; ++i)
                                    if (c0 + i < p.columns) to[i] = Element<T>::from(v[h][i]);
                            }
                        }
                    }
                }
                __syncwarp();   // (the next load of tensor memory is the whole warp's)
            }
            fenceBefore();
            __syncwarp();
            if (lane == 0) barrierArrive(bars + L::DW_EMPTY + acc * 8);
        }
    }
    fenceBefore();
    __syncthreads();
    fenceAfter();
    if (*failed != 0 && warp == 0) {
        copies.land(bars + L::FULL, L::STAGES);
        matricesIn.land(bars + L::W_FULL, 2);
    }
    if (*failed != 0 && warp == 1) {
        mmaCommit<1>(electOne(), bars + L::DRAIN);   // (elects the lane that issued the products)
        if (lane == 0) {
            barrierWait(bars + L::DRAIN, 0);
            atomicOr(p.status, 1);
        }
        __syncwarp();
    }
    if (warp == 1) tmemFree<1>(tmem, L::TMEM);
}

// Joins the partial sums of an expert whose tiles lie in several blocks of the kernel above: thread block b looks after the expert that begins in that
// kernel's block b and goes on behind it, if there is one. `blocks`: blocks of that kernel.
template <class T>
__global__ void __launch_bounds__(256) expert_narrow_join_kernel(const __grid_constant__ ProductArgs p, int blocks, int columns)
{
    chained();
    const int* before = reinterpret_cast<const int*>(p.plan);
    const long long total = before[p.experts];
    const int block = blockIdx.x;
    const int begin = static_cast<int>(total * block / blocks), end = static_cast<int>(total * (block + 1) / blocks);
    if (begin == end || end >= total) return;
    __shared__ int found;
    for (int e = threadIdx.x; e < p.experts; e += 256)   // the expert of tile `end`
        if (before[e] <= end && before[e + 1] > end) found = e;
    __syncthreads();
    const int expert = found;
    if (before[expert] >= end || before[expert] < begin) return;
    // Later blocks with a part of it: with tiles for all blocks every one up to that of its last tile, the first whose end, total * (b + 1) / blocks, reaches
    // before[expert + 1]; with fewer tiles the one block of each tile. (2 or 16 parts read at a time; one expert of 298 rows, 24 -> 64, where a loop over
    // all blocks divided for each, 38 us, so 5 us.)
    const bool full = total >= blocks;
    const int behind = before[expert + 1];
    const int more = full ? static_cast<int>((static_cast<long long>(behind) * blocks + total - 1) / total) - 1 - block : behind - end;
    auto blockOf = [&](int part) { return full ? block + 1 + part : ((end + part + 1) * blocks + static_cast<int>(total) - 1) / static_cast<int>(total) - 1; };
    const int i0 = (blockIdx.y * 256 + threadIdx.x) * 4, n = i0 / columns, c = i0 - n * columns;   // 4 of 128 x columns sums
    if (n < p.sum && c < p.columns) {
        const float* from = p.partial + static_cast<long long>(n) * columns + c;
        float4 sum = *reinterpret_cast<const float4*>(from + (static_cast<long long>(block) * 2 + 1) * 128 * columns);   // the run that block ends with
        int part = 0;                                                                                                    // the runs the later ones begin with
        auto add = [&](auto count) {
            constexpr int N = decltype(count)::value;
            float4 v[N];
#pragma unroll
            for (int k = 0; k < N; ++k)
                v[k] = part + k < more ? *reinterpret_cast<const float4*>(from + static_cast<long long>(blockOf(part + k)) * 2 * 128 * columns) : float4{};
#pragma unroll
            for (int k = 0; k < N; ++k) {
                sum.x += v[k].x;
                sum.y += v[k].y;
                sum.z += v[k].z;
                sum.w += v[k].w;
            }
            part += N;
        };
        while (more - part >= 8) add(std::integral_constant<int, 16>());
        while (part < more) add(std::integral_constant<int, 2>());
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
        T* out = static_cast<T*>(p.out) + (static_cast<long long>(expert) * p.sum + n) * p.columns + c;
        if (p.wideStore) store<T, 4>(out, pack<T, 4>(f));
        else
            for (int k = 0; k < 4 && c + k < p.columns; ++k) out[k] = Element<T>::from(f[k]);
    }
    if (p.gradBias != nullptr && blockIdx.y == 0 && threadIdx.x < p.sum) {
        const float* from = p.partialBias + threadIdx.x;
        float sum = from[(block * 2 + 1) * 128];
#pragma unroll 8
        for (int part = 0; part < more; ++part) sum += from[blockOf(part) * 2 * 128];
        static_cast<T*>(p.gradBias)[static_cast<long long>(expert) * p.sum + threadIdx.x] = Element<T>::from(sum);
    }
}

// Adds up the partial sums of the weight gradients (and, behind the tiles, of the bias gradients) of experts with more than one item. blockIdx.x: tile
// of an expert, blockIdx.y: JOIN_ELEMENTS of it. Most blocks find one item and leave, so there are few of them.
constexpr int JOIN_ELEMENTS = 8192;
template <class T, int BN>
__global__ void __launch_bounds__(256) expert_join_kernel(const __grid_constant__ ProductArgs p)
{
    chained();
    constexpr int ROWS = JOIN_ELEMENTS / BN;
    const int tiles = p.rowTiles * p.columnTiles;
    const int expert = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const int slot = p.plan[expert].x, units = p.plan[expert].y;
    if (units < 2) return;
    const long long unitStride = static_cast<long long>(tiles) * p.tileRows * BN;
    const float* from = p.partial + slot * unitStride + static_cast<long long>(tile) * p.tileRows * BN;
    const int row0 = tile / p.columnTiles * p.tileRows, column0 = tile % p.columnTiles * BN;
    for (int i = threadIdx.x; i < JOIN_ELEMENTS / 4; i += 256) {
        const int r = blockIdx.y * ROWS + i / (BN / 4), c = i % (BN / 4) * 4;
        if (row0 + r >= p.sum || column0 + c >= p.columns) continue;
        float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int u = 0; u < units; ++u) {
            const float4 v = *reinterpret_cast<const float4*>(from + u * unitStride + r * BN + c);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        T* out = static_cast<T*>(p.out) + (static_cast<long long>(expert) * p.sum + row0 + r) * p.outStride + column0 + c;
        const float f[4] = {sum.x, sum.y, sum.z, sum.w};
        if (p.wideStore) store<T, 4>(out, pack<T, 4>(f));
        else
            for (int k = 0; k < 4 && column0 + c + k < p.columns; ++k) out[k] = Element<T>::from(f[k]);
    }
    if (p.gradBias != nullptr && column0 == 0) {
        for (int r = threadIdx.x; r < ROWS; r += 256) {
            const int channel = row0 + blockIdx.y * ROWS + r;
            if (channel >= p.sum || blockIdx.y * ROWS + r >= p.tileRows) break;
            float sum = 0.f;
#pragma unroll 4
            for (int u = 0; u < units; ++u) sum += p.partialBias[static_cast<long long>(slot + u) * p.sum + channel];
            static_cast<T*>(p.gradBias)[static_cast<long long>(expert) * p.sum + channel] = Element<T>::from(sum);
        }
    }
}

// ---- few rows: matrix-vector products -----------------------------------------------------------------------------------------
// The forward product of a handful of rows is bound by reading their experts' matrices once. blockIdx.y is a row; a block of 4 warps takes up
// to 4 consecutive rows of one expert (the first of every 4 does the work) and 16 channels out, 4 per warp, the lanes side by side along the
// channels in. No tiles of 128 rows to fill, no copies where the channels in are odd, and enough blocks to fill the machine.
constexpr int FEW_ROWS = 4, FEW_OUT = 4, FEW_WARPS = 4;
template <class T, int VEC>
__global__ void __launch_bounds__(FEW_WARPS * 32) expert_few_rows_kernel(const __grid_constant__ ExpertArgs a)
{
    chained();
    extern __shared__ __align__(16) float rowsIn[];   // FEW_ROWS x channels in, rounded up to whole accesses of a warp
    __shared__ int found[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y;
    const int n0 = (blockIdx.x * FEW_WARPS + warp) * FEW_OUT;
    if (threadIdx.x == 0) {
        found[0] = a.experts + 1;
        found[1] = 0;
    }
    __syncthreads();
    // the first offset behind the row ends its expert's run (see clampOffset): that expert is the one before it
    int behind = a.experts + 1;
    for (int e = threadIdx.x; e <= a.experts; e += FEW_WARPS * 32)
        if (a.offsets[e] > row) { behind = e; break; }
    if (behind <= a.experts) atomicMin(&found[0], behind);
    __syncthreads();
    behind = found[0];
    T* y = static_cast<T*>(a.y.data);
    if (behind == 0 || behind > a.experts) {   // nobody's row
        for (int n = n0 + lane; n < min(n0 + FEW_OUT, a.channelsOut); n += 32) y[row * a.y.stride + n] = Element<T>::from(0.f);
        return;
    }
    int begin = 0;
    for (int e = threadIdx.x; e < behind; e += FEW_WARPS * 32) begin = max(begin, a.offsets[e]);
    if (begin > 0) atomicMax(&found[1], begin);
    __syncthreads();
    begin = found[1];
    const int expert = behind - 1, end = static_cast<int>(min(a.rows, static_cast<long long>(a.offsets[behind])));
    if ((row - begin) % FEW_ROWS != 0) return;
    const int count = min(FEW_ROWS, end - row);
    const int stride = (a.channelsIn + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
    for (int r = 0; r < count; ++r) {
        const T* x = static_cast<const T*>(a.x.data) + (row + r) * a.x.stride;
        for (int k = threadIdx.x; k < stride; k += FEW_WARPS * 32) rowsIn[r * stride + k] = k < a.channelsIn ? Element<T>::to(x[k]) : 0.f;
    }
    __syncthreads();
    const T* w = static_cast<const T*>(a.weight) + (static_cast<long long>(expert) * a.channelsOut + n0) * a.channelsIn;
    float sum[FEW_OUT][FEW_ROWS] = {};
    auto step = [&](int k0, auto unroll) {
        constexpr int U = decltype(unroll)::value;
        Pack<T, VEC> v[U][FEW_OUT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int o = 0; o < FEW_OUT; ++o) {
                const int k = k0 + (u * 32 + lane) * VEC;
                v[u][o] = {};
                if (k < a.channelsIn && n0 + o < a.channelsOut) v[u][o] = load<T, VEC>(w + static_cast<long long>(o) * a.channelsIn + k);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + (u * 32 + lane) * VEC;
            float f[FEW_OUT][VEC];
#pragma unroll
            for (int o = 0; o < FEW_OUT; ++o) unpack<T, VEC>(v[u][o], f[o]);
#pragma unroll
            for (int r = 0; r < FEW_ROWS; ++r) {
                if (r >= count) break;
                float x[VEC];
                if constexpr (VEC % 4 == 0) {
#pragma unroll
                    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(&x[i]) = *reinterpret_cast<const float4*>(rowsIn + r * stride + k + i);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[i] = rowsIn[r * stride + k + i];
                }
#pragma unroll
                for (int o = 0; o < FEW_OUT; ++o)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) sum[o][r] = fmaf(f[o][i], x[i], sum[o][r]);
            }
        }
    };
    int k0 = 0;
    for (; k0 + 4 * 32 * VEC <= stride; k0 += 4 * 32 * VEC) step(k0, std::integral_constant<int, 4>());
    for (; k0 < stride; k0 += 32 * VEC) step(k0, std::integral_constant<int, 1>());
#pragma unroll
    for (int o = 0; o < FEW_OUT; ++o)
#pragma unroll
        for (int r = 0; r < FEW_ROWS; ++r) {
            if (r >= count) break;
            const float all = groupSum<32>(sum[o][r]);
            if (lane == 0 && n0 + o < a.channelsOut) {
                const float b = a.bias != nullptr ? Element<T>::to(static_cast<const T*>(a.bias)[static_cast<long long>(expert) * a.channelsOut + n0 + o]) : 0.f;
                y[(row + r) * a.y.stride + n0 + o] = Element<T>::from(all + b);
            }
        }
}

// ---- bias gradient without a weight gradient: column sums of an expert's rows ----------------------------------------------------
// blockIdx.x: expert, blockIdx.y: 32 x 8 columns. 8 warps take strided rows, then join.
template <class T>
__global__ void __launch_bounds__(256) expert_bias_kernel(const __grid_constant__ ProductArgs p, const T* __restrict__ dy, long long stride, T* __restrict__ out)
{
    chained();
    __shared__ float shared[8][32];
    __shared__ int reached[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.y * 32 + lane;
    int begin = 0;
    for (int e = threadIdx.x; e <= static_cast<int>(blockIdx.x); e += 256) begin = max(begin, clampOffset(p, e));
    begin = __reduce_max_sync(0xffffffffu, begin);
    if (lane == 0) reached[warp] = begin;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) begin = max(begin, reached[w]);
    const int end = max(begin, clampOffset(p, blockIdx.x + 1));
    float sum = 0.f;
    if (c < p.columns) {
#pragma unroll 8
        for (int r = begin + warp; r < end; r += 8) sum += Element<T>::to(dy[r * stride + c]);
    }
    shared[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.columns) {
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += shared[w][lane];
        out[static_cast<long long>(blockIdx.x) * p.columns + c] = Element<T>::from(sum);
    }
}

// ---- copies of operands the TMA cannot read --------------------------------------------------------------------------------
// rows of `columns` elements -> rows of `padded` (a multiple of 8) elements, zeros behind. A thread puts 8 elements together from reads of WORD elements
// (2 where the rows begin on 4 bytes), for PAD_ROWS rows, `pass` rows apart. With `offsets`, rows of an expert without rows of x, which no product reads, are
// left out. 36838 rows of 690 bfloat16: 27 us (element by element, which divides for each, 60 us).
constexpr int PAD_ROWS = 4;
template <class T, int WORD>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T* __restrict__ in, long long stride, T* __restrict__ out, long long rows, int columns, int pieces, int pass,
                                                       const int* __restrict__ offsets, int perExpert)
{
    chained();
    const int rowInPass = pass == 1 ? 0 : static_cast<int>(threadIdx.x) / pieces, piece = blockIdx.y * 256 + (pass == 1 ? threadIdx.x : threadIdx.x - rowInPass * pieces);
    if (rowInPass >= pass || piece >= pieces) return;
    const int c = piece * 8;
    const long long first = static_cast<long long>(blockIdx.x) * (pass * PAD_ROWS) + rowInPass;
    bool copy[PAD_ROWS];
    Pack<T, 8> v[PAD_ROWS];
#pragma unroll
    for (int k = 0; k < PAD_ROWS; ++k) {
        const long long r = first + k * pass;
        copy[k] = r < rows;
        if (copy[k] && offsets != nullptr) {
            const int e = static_cast<int>(r / perExpert);
            copy[k] = offsets[e + 1] > offsets[e];
        }
    }
#pragma unroll
    for (int k = 0; k < PAD_ROWS; ++k) {
        const T* from = in + (first + k * pass) * stride + c;
#pragma unroll
        for (int i = 0; i < 8; i += WORD) {
            Pack<T, WORD> w = {};
            if (copy[k] && c + i < columns) w = load<T, WORD>(from + i);
#pragma unroll
            for (int j = 0; j < WORD; ++j) v[k].v[i + j] = w.v[j];
        }
    }
#pragma unroll
    for (int k = 0; k < PAD_ROWS; ++k)
        if (copy[k]) store<T, 8>(out + ((first + k * pass) * pieces + piece) * 8, v[k]);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder()
{
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}
// matrix of `rows` x `columns` 16-bit elements (`matrices` of them, one behind the other, for a 3-D map), boxes of 64 x 64
cudaError_t encodeMap(CUtensorMap& map, int type, const void* data, long long matrices, long long rows, int columns, long long stride)
{
    const EncodeFn encode = encoder();
    if (encode == nullptr) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(matrices)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride) * 2, static_cast<cuuint64_t>(stride) * 2 * rows};
    const cuuint32_t box[3] = {64, 64, 1}, one[3] = {1, 1, 1};
    auto run = [&] {
        return encode(&map, type == TYPE_HALF ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, matrices > 0 ? 3 : 2, const_cast<void*>(data), dims,
                      strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = run();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {   // a thread's first call (a backward pass runs in a thread of its own): the driver wants a context, which the runtime binds
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaSetDevice(device);
        if (e != cudaSuccess) return e;
        r = run();
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }
int pad8(int n) { return (n + 7) / 8 * 8; }
// rows the TMA can read where they lie
bool direct(const void* data, long long stride, int columns) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && stride % 8 == 0 && stride >= columns; }

// Shape of the tiles. Pairs of blocks (256 x 256) read a third less shared memory per product, but cut rows into coarser pieces: taken where
// D is wide and an expert has rows enough for two such tiles on average.
struct Shape {
    int width, ctas;
};
Shape shapeOf(long long rows, int columns)
{
    if (columns <= 64) return {64, 1};
    if (columns <= 128) return {128, 1};
    return {256, rows >= 512 ? 2 : 1};
}
Shape rowShape(const ExpertArgs& a, int columns) { return shapeOf(a.rows / a.experts, columns); }                       // forward, input gradient
Shape weightShape(const ExpertArgs& a) { return shapeOf(a.channelsOut > 128 ? 512 : 0, a.channelsIn); }                 // weight gradient

// Rows per item of the weight gradient. Cutting an expert's rows fills the blocks where its tiles alone do not, at the price of a write and
// a read of an fp32 tile per item. The estimate below weighs the two for runs of average length: a step of 64 rows takes about 0.3 us
// (256 x 256 tiles at the tensor core's rate, narrow ones at the memory's), partial sums move at about 5 TB/s. 64 experts of 4096 rows of
// 256 x 256: whole runs 49 us, cut into 320 items 74 us and 44 us for their sums. An expert with more than twice the average is cut in any case, or with
// more than a sixth of a block's share of all steps where that is later (a quarter cost 64 experts of 1024 x 1024, one with 8 times the rows of the others, 154
// us for 148): every item that may be cut wants an fp32 tile of scratch, and with the shares in mind their number goes with the blocks (12 tiles of a block and no
// more, 230 MB), not with the experts. 65536 rows are cut in any case: tensor
// memory cuts its sums off instead of rounding them, and a sum of one sign comes out too small, by 1.0e-4 of itself over 16384 rows and 3.9e-4, less than
// half a unit of half's last place, over 65536.
int weightChunk(const ExpertArgs& a, int tiles, int tileElements, int blocks)
{
    const double run = static_cast<double>(a.rows) / a.experts;
    double best = 0;
    int pieces = 1;
    for (int k = 1; k <= 1024 && (k == 1 || run / k >= 256); k *= 2) {
        const double items = static_cast<double>(a.experts) * k * tiles;
        const double time = std::ceil(items / blocks) * std::ceil(run / k / BK) * 0.3 + (k > 1 ? 5.0 + items * tileElements * 8 / 5e6 : 0.0);
        if (k == 1 || time < best) {
            best = time;
            pieces = k;
        }
    }
    const double rows = pieces == 1 ? run * std::max(2.0, static_cast<double>(a.experts) * tiles / blocks / 6) : run / pieces;
    return static_cast<int>(std::min<double>(std::max<double>(std::ceil(rows / BK) * BK, 512), 1 << 16));
}

// scratch: [x | weight | dy in a form the TMA reads, where needed | partial sums of the weight and bias gradients | their plan]
struct Scratch {
    size_t x, weight, gradY, partial, partialBias, plan, bytes;
    bool narrow;   // both gradients in one pass
    int chunk, rowTiles, columnTiles, tileRows;
    Shape shape;
    Scratch(const ExpertArgs& a, bool adjoint)
    {
        const bool forward = !adjoint;
        const size_t rows = static_cast<size_t>(a.rows), matrices = static_cast<size_t>(a.experts) * a.channelsOut;
        bytes = 0;
        auto take = [&](bool needed, size_t n) {
            const size_t at = bytes;
            if (needed) bytes += align256(n);
            return at;
        };
        const bool weights = adjoint && a.gradWeight != nullptr;
        x = take((forward || weights) && !direct(a.x.data, a.x.stride, a.channelsIn), rows * pad8(a.channelsIn) * 2);
        weight = take((forward || a.gradX.data != nullptr) && !direct(a.weight, a.channelsIn, a.channelsIn), matrices * pad8(a.channelsIn) * 2);
        gradY = take(adjoint && !direct(a.gradY.data, a.gradY.stride, a.channelsOut), rows * pad8(a.channelsOut) * 2);
        shape = weightShape(a);
        tileRows = BM * shape.ctas;
        rowTiles = (a.channelsOut + tileRows - 1) / tileRows;
        columnTiles = (a.channelsIn + shape.width - 1) / shape.width;
        const int tiles = rowTiles * columnTiles;
        chunk = weightChunk(a, tiles, tileRows * shape.width, a.numSMs / shape.ctas);
        narrow = weights && a.gradX.data != nullptr && a.channelsIn <= 128 && a.channelsOut <= 128;
        if (narrow) {
            const size_t slots = static_cast<size_t>(a.numSMs) * 2 * 128;
            partial = take(true, slots * (a.channelsIn <= 64 ? 64 : 128) * 4);
            partialBias = take(true, slots * 4);
            plan = take(true, (static_cast<size_t>(a.experts) + 1) * 4);
            return;
        }
        // slots: items of the runs that are cut, which have at least chunk + 1 rows each
        const size_t cut = std::min<size_t>(a.experts, rows / (static_cast<size_t>(chunk) + 1)), slots = cut > 0 ? rows / chunk + cut : 0;
        partial = take(weights, slots * tiles * tileRows * shape.width * 4);
        partialBias = take(weights, slots * a.channelsOut * 4);
        plan = take(weights && slots > 0, static_cast<size_t>(a.experts) * sizeof(int2));
    }
};

// `offsets`: of experts with `perExpert` rows of the matrix each, or null
template <class T>
cudaError_t readable(const void*& data, long long& stride, long long rows, int columns, void* scratch, cudaStream_t stream, const int* offsets = nullptr, int perExpert = 1)
{
    if (direct(data, stride, columns)) return cudaSuccess;
    const int pieces = pad8(columns) / 8, pass = pieces > 128 ? 1 : 256 / pieces;
    const dim3 grid(static_cast<unsigned>((rows + pass * PAD_ROWS - 1) / (pass * PAD_ROWS)), pass == 1 ? (pieces + 255) / 256 : 1);
    const bool pairs = columns % 2 == 0 && stride % 2 == 0 && reinterpret_cast<uintptr_t>(data) % 4 == 0;
    launchChained(pairs ? pad_rows_kernel<T, 2> : pad_rows_kernel<T, 1>, grid, 256, 0, stream, 1, static_cast<const T*>(data), stride, static_cast<T*>(scratch), rows, columns, pieces,
                  pass, offsets, perExpert);
    data = scratch;
    stride = pieces * 8;
    return cudaGetLastError();
}

template <class T, int MODE, int BN, int CTAS, bool SUMS>
cudaError_t launchProduct(const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& p, int numSMs, cudaStream_t stream)
{
    auto* kernel = expert_product_kernel<T, MODE, BN, CTAS, SUMS>;
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), Layout<BN, CTAS>::bytes(EXPERTS_MAX));
    if (e != cudaSuccess) return e;
    return launchChained(kernel, numSMs / CTAS * CTAS, blockThreads(SUMS), Layout<BN, CTAS>::bytes(p.experts), stream, CTAS, a, b, p);
}
template <class T, int MODE, bool SUMS = false>
cudaError_t launchShape(const Shape& shape, const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& p, int numSMs, cudaStream_t stream)
{
    if (shape.width == 64) return launchProduct<T, MODE, 64, 1, SUMS>(a, b, p, numSMs, stream);
    if (shape.width == 128) return launchProduct<T, MODE, 128, 1, SUMS>(a, b, p, numSMs, stream);
    if (shape.ctas == 1) return launchProduct<T, MODE, 256, 1, SUMS>(a, b, p, numSMs, stream);
    return launchProduct<T, MODE, 256, 2, SUMS>(a, b, p, numSMs, stream);
}

ProductArgs common(const ExpertArgs& a)
{
    ProductArgs p{};
    p.rows = a.rows;
    p.experts = a.experts;
    p.offsets = a.offsets;
    p.status = a.status;
    return p;
}
bool wideOut(const void* out, long long stride, int columns) { return (reinterpret_cast<uintptr_t>(out) & 15) == 0 && stride % 8 == 0 && columns % 8 == 0; }

// Rows that the matrix-vector kernel takes. Its time goes with the rows, the tensor kernel's hardly; half, us of the two, back to back: 64 experts of
// 1024 -> 2048, 2 rows 3.6 / 10.6, 16 rows 12.0 / 13.1, 24 rows 21 / 20, 32 rows 31 / 26; 16 experts of 1024 -> 1024, 32 rows 11.8 / 11.7, 64 rows 21 / 11;
// 512 experts of 256 -> 256, 64 rows 6.0 / 9.1; 128 experts of 512 -> 2048, 16 rows 10.5 / 9.8, 32 rows 22 / 13, 64 rows 39 / 16; one of 4096 -> 4096, 2 rows
// 11 / 24, 4 rows (which share their reads) 18 / 24.
bool fewRows(const ExpertArgs& a)
{
    return a.rows <= 64 && a.rows * a.channelsIn * a.channelsOut <= 1ll << (a.rows <= FEW_ROWS ? 26 : 25) && FEW_ROWS * (a.channelsIn + 256) * 4 <= 200 * 1024;
}

template <class T>
cudaError_t forwardFewRows(const ExpertArgs& a, cudaStream_t stream)
{
    const dim3 grid((a.channelsOut + FEW_WARPS * FEW_OUT - 1) / (FEW_WARPS * FEW_OUT), static_cast<unsigned>(a.rows));
    const bool vec = (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0 && a.channelsIn % 8 == 0;
    auto go = [&](auto* kernel, int width) {
        const int bytes = FEW_ROWS * ((a.channelsIn + 32 * width - 1) / (32 * width) * (32 * width)) * 4;
        if (bytes > 47 * 1024) {   // (48 KB without asking, which the kernel's static shared memory counts towards)
            const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), 200 * 1024);
            if (e != cudaSuccess) return e;
        }
        launchChained(kernel, grid, FEW_WARPS * 32, bytes, stream, 1, a);
        return cudaGetLastError();
    };
    return vec ? go(expert_few_rows_kernel<T, 8>, 8) : go(expert_few_rows_kernel<T, 1>, 1);
}

template <class T>
cudaError_t forward(const ExpertArgs& a, cudaStream_t stream)
{
    if (fewRows(a)) return forwardFewRows<T>(a, stream);
    const Scratch s(a, false);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    const void *x = a.x.data, *w = a.weight;
    long long xStride = a.x.stride, wStride = a.channelsIn;
    cudaError_t e = readable<T>(x, xStride, a.rows, a.channelsIn, base + s.x, stream);
    if (e == cudaSuccess) e = readable<T>(w, wStride, static_cast<long long>(a.experts) * a.channelsOut, a.channelsIn, base + s.weight, stream, a.offsets, a.channelsOut);
    CUtensorMap mapX, mapW;
    if (e == cudaSuccess) e = encodeMap(mapX, a.type, x, 0, a.rows, a.channelsIn, xStride);
    if (e == cudaSuccess) e = encodeMap(mapW, a.type, w, a.experts, a.channelsOut, a.channelsIn, wStride);
    if (e != cudaSuccess) return e;
    ProductArgs p = common(a);
    p.columns = a.channelsOut;
    p.sum = a.channelsIn;
    const Shape shape = rowShape(a, p.columns);
    p.columnTiles = (p.columns + shape.width - 1) / shape.width;
    p.tileRows = BM * shape.ctas;
    p.out = a.y.data;
    p.outStride = a.y.stride;
    p.bias = a.bias;
    p.wideStore = wideOut(p.out, p.outStride, p.columns);
    return launchShape<T, FORWARD>(shape, mapX, mapW, p, a.numSMs, stream);
}

template <class T, int NB, int KB>
cudaError_t launchNarrow(const CUtensorMap& y, const CUtensorMap& x, const CUtensorMap& w, const ProductArgs& p, const ExpertArgs& a, cudaStream_t stream)
{
    auto go = [&](auto* kernel) {
        const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), NarrowLayout<NB, KB>::bytes(EXPERTS_MAX));
        if (e != cudaSuccess) return e;
        launchChained(kernel, a.numSMs, blockThreads(true), NarrowLayout<NB, KB>::bytes(a.experts), stream, 1, y, x, w, p, static_cast<T*>(a.gradX.data), a.gradX.stride, wideOut(a.gradX.data, a.gradX.stride, a.channelsIn));
        return cudaGetLastError();
    };
    cudaError_t e = a.gradBias != nullptr ? go(expert_narrow_adjoint_kernel<T, NB, KB, true>) : go(expert_narrow_adjoint_kernel<T, NB, KB, false>);
    if (e != cudaSuccess) return e;
    launchChained(expert_narrow_join_kernel<T>, dim3(a.numSMs, (a.channelsOut * KB * 64 + 1023) / 1024), 256, 0, stream, 1, p, a.numSMs, KB * 64);
    return cudaGetLastError();
}

template <class T>
cudaError_t adjoint(const ExpertArgs& a, cudaStream_t stream)
{
    const Scratch s(a, true);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    cudaError_t e = cudaSuccess;
    if (a.gradBias != nullptr && (a.gradWeight == nullptr || a.rows == 0)) {
        ProductArgs p = common(a);
        p.columns = a.channelsOut;
        launchChained(expert_bias_kernel<T>, dim3(a.experts, (a.channelsOut + 31) / 32), 256, 0, stream, 1, p, static_cast<const T*>(a.gradY.data), a.gradY.stride, static_cast<T*>(a.gradBias));
        e = cudaGetLastError();
    }
    if (a.rows == 0) {
        if (e == cudaSuccess && a.gradWeight != nullptr)
            e = cudaMemsetAsync(a.gradWeight, 0, static_cast<size_t>(a.experts) * a.channelsOut * a.channelsIn * 2, stream);
        return e;
    }
    const void *x = a.x.data, *w = a.weight, *dy = a.gradY.data;
    long long xStride = a.x.stride, wStride = a.channelsIn, dyStride = a.gradY.stride;
    CUtensorMap mapX, mapW, mapY;
    if (e == cudaSuccess) e = readable<T>(dy, dyStride, a.rows, a.channelsOut, base + s.gradY, stream);
    if (e == cudaSuccess) e = encodeMap(mapY, a.type, dy, 0, a.rows, a.channelsOut, dyStride);
    if (e == cudaSuccess && s.narrow) {
        e = readable<T>(w, wStride, static_cast<long long>(a.experts) * a.channelsOut, a.channelsIn, base + s.weight, stream, a.offsets, a.channelsOut);
        if (e == cudaSuccess) e = readable<T>(x, xStride, a.rows, a.channelsIn, base + s.x, stream);
        if (e == cudaSuccess) e = encodeMap(mapW, a.type, w, a.experts, a.channelsOut, a.channelsIn, wStride);
        if (e == cudaSuccess) e = encodeMap(mapX, a.type, x, 0, a.rows, a.channelsIn, xStride);
        if (e != cudaSuccess) return e;
        ProductArgs p = common(a);
        p.columns = a.channelsIn;
        p.sum = a.channelsOut;
        p.tileRows = BM;
        p.out = a.gradWeight;
        p.gradBias = a.gradBias;
        p.partial = reinterpret_cast<float*>(base + s.partial);
        p.partialBias = reinterpret_cast<float*>(base + s.partialBias);
        p.plan = reinterpret_cast<int2*>(base + s.plan);
        p.wideStore = wideOut(a.gradWeight, a.channelsIn, a.channelsIn);
        if (a.channelsOut <= 64) return a.channelsIn <= 64 ? launchNarrow<T, 1, 1>(mapY, mapX, mapW, p, a, stream) : launchNarrow<T, 1, 2>(mapY, mapX, mapW, p, a, stream);
        return a.channelsIn <= 64 ? launchNarrow<T, 2, 1>(mapY, mapX, mapW, p, a, stream) : launchNarrow<T, 2, 2>(mapY, mapX, mapW, p, a, stream);
    }
    if (e == cudaSuccess && a.gradX.data != nullptr) {
        e = readable<T>(w, wStride, static_cast<long long>(a.experts) * a.channelsOut, a.channelsIn, base + s.weight, stream, a.offsets, a.channelsOut);
        if (e == cudaSuccess) e = encodeMap(mapW, a.type, w, a.experts, a.channelsOut, a.channelsIn, wStride);
        if (e != cudaSuccess) return e;
        ProductArgs p = common(a);
        p.columns = a.channelsIn;
        p.sum = a.channelsOut;
        const Shape shape = rowShape(a, p.columns);
        p.columnTiles = (p.columns + shape.width - 1) / shape.width;
        p.tileRows = BM * shape.ctas;
        p.out = a.gradX.data;
        p.outStride = a.gradX.stride;
        p.wideStore = wideOut(p.out, p.outStride, p.columns);
        e = launchShape<T, INPUT>(shape, mapY, mapW, p, a.numSMs, stream);
    }
    if (e == cudaSuccess && a.gradWeight != nullptr) {
        e = readable<T>(x, xStride, a.rows, a.channelsIn, base + s.x, stream);
        if (e == cudaSuccess) e = encodeMap(mapX, a.type, x, 0, a.rows, a.channelsIn, xStride);
        if (e != cudaSuccess) return e;
        ProductArgs p = common(a);
        p.columns = a.channelsIn;
        p.sum = a.channelsOut;
        p.rowTiles = s.rowTiles;
        p.columnTiles = s.columnTiles;
        p.chunk = s.chunk;
        p.out = a.gradWeight;
        p.outStride = a.channelsIn;
        p.partial = reinterpret_cast<float*>(base + s.partial);
        p.plan = a.rows > s.chunk ? reinterpret_cast<int2*>(base + s.plan) : nullptr;
        p.wideStore = wideOut(p.out, p.outStride, p.columns);
        p.tileRows = s.tileRows;
        p.gradBias = a.gradBias;
        p.partialBias = reinterpret_cast<float*>(base + s.partialBias);
        e = a.gradBias != nullptr ? launchShape<T, WEIGHTS, true>(s.shape, mapY, mapX, p, a.numSMs, stream)
                                  : launchShape<T, WEIGHTS, false>(s.shape, mapY, mapX, p, a.numSMs, stream);
        if (e == cudaSuccess && a.rows > s.chunk) {
            const dim3 grid(a.experts * s.rowTiles * s.columnTiles, s.tileRows * s.shape.width / JOIN_ELEMENTS);
            if (s.shape.width == 64) launchChained(expert_join_kernel<T, 64>, grid, 256, 0, stream, 1, p);
            else if (s.shape.width == 128) launchChained(expert_join_kernel<T, 128>, grid, 256, 0, stream, 1, p);
            else launchChained(expert_join_kernel<T, 256>, grid, 256, 0, stream, 1, p);
            e = cudaGetLastError();
        }
    }
    return e;
}

} // namespace

size_t expertBytes(const ExpertArgs& a, bool adjoint) { return a.rows == 0 || (!adjoint && fewRows(a)) ? 0 : Scratch(a, adjoint).bytes; }

cudaError_t launchExpertForward(const ExpertArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return a.type == TYPE_HALF ? forward<__half>(a, stream) : forward<__nv_bfloat16>(a, stream);
}
cudaError_t launchExpertAdjoint(const ExpertArgs& a, cudaStream_t stream)
{
    return a.type == TYPE_HALF ? adjoint<__half>(a, stream) : adjoint<__nv_bfloat16>(a, stream);
}

} // namespace kernel
} // namespace qmlp
