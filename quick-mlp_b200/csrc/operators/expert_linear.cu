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
// One persistent block per SM: a TMA warp, an MMA warp, four epilogue warps; a ring of operand stages between the first two, two
// accumulators between the last two, so that the products of a tile run under the epilogue of the one before. Which tile is
// whose follows from the offsets, which every block adds up for itself: the group sizes never travel to the host.
// Waits are bounded: on a timeout the block drains, gives its tensor memory back and sets the library's status word.
#include "common.cuh"

#include <algorithm>
#include <type_traits>

#include <cuda.h>

namespace qmlp {
namespace kernel {
namespace {

using namespace ops;

// ---- PTX ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tmaLoad2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tmaLoad3(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void fenceProxyAsync() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(static_cast<uint32_t>(accumulate)) : "memory");
}
__device__ __forceinline__ void mmaCommit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 consecutive fp32 columns of this thread's lane of tensor memory
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
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// descriptor of a 128-byte swizzled operand: groups of 8 rows of 128 bytes lie 1024 bytes apart. K-major: the rows are rows of the
// operand. MN-major: the rows run along the sum, and blocks of 64 rows of the operand lie `lead` bytes apart.
__device__ __forceinline__ uint64_t operandDescriptor(uint32_t address, uint32_t lead)
{
    return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// ---- plan ------------------------------------------------------------------------------------------------------------------
enum Product : int { FORWARD = 0, INPUT = 1, WEIGHTS = 2 };
constexpr int BM = 128, BK = 64, BOX = 64 * 128;   // tile of D, block along the sum, bytes of a box of 64 x 64 elements
constexpr int EPILOGUE_WARPS = 4, BLOCK = (2 + EPILOGUE_WARPS) * 32;

template <int BN>
struct Layout {
    static constexpr int ABYTES = BM * 128, BBYTES = BN * 128, STAGE = ABYTES + BBYTES;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int ACC = BN;                    // columns of an accumulator
    static constexpr int TMEM = 2 * ACC < 32 ? 32 : 2 * ACC;
    static constexpr int OUT = EPILOGUE_WARPS * 32 * 128;   // 32 rows x 64 elements of 16 bits per epilogue warp
    static constexpr int BARS = 16 * 8 + 4 * 8 + 32;
    // 1 KB for the alignment of the ring
    static constexpr int bytes(int experts) { return 1024 + STAGES * STAGE + OUT + BARS + 2 * (experts + 1) * 4; }
};

struct ProductArgs {
    long long rows;
    int experts, columns, sum;    // columns of D; length of the sum (forward, input), channels out (weights)
    int rowTiles, columnTiles;    // weights: tiles of D; else columnTiles alone
    int chunk;                    // weights: rows of an expert per item
    const int* offsets;
    void* out;
    long long outStride;          // elements between rows of D in memory
    const void* bias;             // forward: (experts, columns) or null
    int* plan;                    // weights: units of the experts before, written for the join; null where no expert can have two
    float* partial;               // weights: items x tiles x 128 x BN sums of experts with more than one item
    int* status;
    bool wideStore;               // rows of D can be written 16 bytes at a time
};

// Offsets are taken as the running maximum of what they say, within [0, rows]: runs are disjoint whatever the caller's array holds.
__device__ __forceinline__ int clampOffset(const ProductArgs& p, int e)
{
    return static_cast<int>(max(0ll, min(p.rows, static_cast<long long>(p.offsets[e]))));
}
// units of work along `rows` rows of an expert
template <int MODE>
__device__ __forceinline__ int unitsOf(const ProductArgs& p, int rows)
{
    return MODE == WEIGHTS ? max(1, (rows + p.chunk - 1) / p.chunk) : (rows + BM - 1) / BM;
}
// One warp: bounds[e] = first row of expert e, bounds[experts] the end of the last one; before[e] = units of the experts before.
template <int MODE>
__device__ __forceinline__ void planExperts(const ProductArgs& p, int* bounds, int* before)
{
    const int lane = threadIdx.x & 31;
    int reached = clampOffset(p, 0), carry = 0;
    if (lane == 0) {
        bounds[0] = reached;
        before[0] = 0;
    }
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
        const int e = e0 + lane;
        int end = e < p.experts ? clampOffset(p, e + 1) : 0;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end = max(end, up);
        }
        end = max(end, reached);
        const int left = __shfl_up_sync(0xffffffffu, end, 1), begin = lane == 0 ? reached : left;
        int units = e < p.experts ? unitsOf<MODE>(p, end - begin) : 0;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, units, o);
            if (lane >= o) units += up;
        }
        if (e < p.experts) {
            bounds[e + 1] = end;
            before[e + 1] = carry + units;
        }
        reached = __shfl_sync(0xffffffffu, end, 31);
        carry += __shfl_sync(0xffffffffu, units, 31);
    }
}

// One tile of D: its expert, the run of rows it reads (forward, input: its own rows) and where it lies.
struct Tile {
    int expert, unit, units, begin, end, row, column;
};
// Walks the tiles of a block. All threads of a warp call next() together: 32 experts are looked at in one step.
template <int MODE, int BN>
struct Walk {
    const ProductArgs& p;
    const int *bounds, *before;   // planExperts
    long long tile;
    int expert = 0;
    __device__ __forceinline__ Walk(const ProductArgs& args, const int* rows, const int* units) : p(args), bounds(rows), before(units), tile(blockIdx.x) {}
    __device__ __forceinline__ bool next(Tile& t)
    {
        const long long perUnit = MODE == WEIGHTS ? static_cast<long long>(p.rowTiles) * p.columnTiles : p.columnTiles;
        if (tile >= before[p.experts] * perUnit) return false;
        const int unit = static_cast<int>(tile / perUnit), at = static_cast<int>(tile - unit * perUnit);
        const int lane = threadIdx.x & 31;
        for (;;) {   // first expert whose units reach behind `unit`
            const int e = expert + 1 + lane;
            const unsigned passed = __ballot_sync(0xffffffffu, e <= p.experts && before[e] <= unit);
            expert += __popc(passed);
            if (passed != 0xffffffffu) break;
        }
        const int first = bounds[expert], last = bounds[expert + 1];
        t.expert = expert;
        t.unit = unit - before[expert];
        t.units = before[expert + 1] - before[expert];
        if constexpr (MODE == WEIGHTS) {
            t.begin = first + t.unit * p.chunk;
            t.end = min(last, t.begin + p.chunk);
            t.row = at / p.columnTiles * BM;
            t.column = at % p.columnTiles * BN;
        } else {
            t.begin = first + t.unit * BM;
            t.end = min(last, t.begin + BM);
            t.row = t.begin;
            t.column = at * BN;
        }
        tile += gridDim.x;
        return true;
    }
    // blocks along the sum
    __device__ __forceinline__ int steps(const Tile& t) const { return MODE == WEIGHTS ? (t.end - t.begin + BK - 1) / BK : (p.sum + BK - 1) / BK; }
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

// operand format in the instruction descriptor
template <class T> constexpr uint32_t FORMAT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;

template <class T, int MODE, int BN>
__global__ void __launch_bounds__(BLOCK, 1)
    expert_product_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ ProductArgs p)
{
    using L = Layout<BN>;
    extern __shared__ unsigned char dynamic[];
    const uint32_t raw = smemAddress(dynamic), ring = (raw + 1023u) & ~1023u;
    unsigned char* base = dynamic + (ring - raw);
    unsigned char* outStage = base + L::STAGES * L::STAGE;
    const uint32_t bars = ring + L::STAGES * L::STAGE + L::OUT;
    const uint32_t full = bars, empty = bars + 8 * 8, accFull = bars + 16 * 8, accEmpty = accFull + 16, drain = bars + 16 * 8 + 4 * 8 + 16;
    volatile int* failed = reinterpret_cast<volatile int*>(outStage + L::OUT + 16 * 8 + 4 * 8);
    uint32_t* tmemBase = reinterpret_cast<uint32_t*>(outStage + L::OUT + 16 * 8 + 4 * 8 + 8);
    int *bounds = reinterpret_cast<int*>(outStage + L::OUT + L::BARS), *before = bounds + p.experts + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            barrierInit(full + s * 8, 1);
            barrierInit(empty + s * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrierInit(accFull + i * 8, 1);
            barrierInit(accEmpty + i * 8, EPILOGUE_WARPS);
        }
        barrierInit(drain, 1);
        *failed = 0;
        barrierInitDone();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smemAddress(tmemBase)), "r"(L::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2) planExperts<MODE>(p, bounds, before);
    fenceBefore();
    __syncthreads();
    fenceAfter();
    const uint32_t tmem = *tmemBase;
    if (MODE == WEIGHTS && p.plan != nullptr && blockIdx.x == 0)   // for the kernel that joins the partial sums
        for (int e = threadIdx.x; e <= p.experts; e += BLOCK) p.plan[e] = before[e];
    Walk<MODE, BN> walk(p, bounds, before);
    Tile t;

    if (warp == 0) {
        // ---- operands -------------------------------------------------------------------------------------------------
        uint32_t stage = 0, phase = 0;
        long long issued = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            const int steps = walk.steps(t);
            for (int k = 0; k < steps; ++k) {
                if (!await(empty + stage * 8, phase ^ 1, failed)) { ok = false; break; }
                if (lane == 0) {
                    const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES, bar = full + stage * 8;
                    barrierExpect(bar, L::STAGE);
                    if constexpr (MODE == WEIGHTS) {
                        const int row = t.begin + k * BK;
#pragma unroll
                        for (int i = 0; i < BM / 64; ++i) tmaLoad2(a + i * BOX, &mapA, t.row + i * 64, row, bar);
#pragma unroll
                        for (int i = 0; i < BN / 64; ++i) tmaLoad2(b + i * BOX, &mapB, t.column + i * 64, row, bar);
                    } else {
#pragma unroll
                        for (int i = 0; i < BM / 64; ++i) tmaLoad2(a + i * BOX, &mapA, k * BK, t.begin + i * 64, bar);
#pragma unroll
                        for (int i = 0; i < BN / 64; ++i) {
                            if constexpr (MODE == FORWARD) tmaLoad3(b + i * BOX, &mapB, k * BK, t.column + i * 64, t.expert, bar);
                            else tmaLoad3(b + i * BOX, &mapB, t.column + i * 64, k * BK, t.expert, bar);
                        }
                    }
                }
                __syncwarp();
                ++issued;
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        if (!ok) {   // copies in flight land before the block's shared memory is given back
            const int outstanding = static_cast<int>(min(issued, static_cast<long long>(L::STAGES)));
            for (int i = 0; i < outstanding; ++i) {
                if (stage == 0) { stage = L::STAGES; phase ^= 1; }
                --stage;
                for (uint32_t n = 0; n < WAIT_LIMIT && !barrierTest(full + stage * 8, phase); ++n) {}
            }
        }
    } else if (warp == 1) {
        // ---- products -------------------------------------------------------------------------------------------------
        constexpr uint32_t instruction = (1u << 4) | (FORMAT<T> << 7) | (FORMAT<T> << 10) | (MODE == WEIGHTS ? 1u << 15 : 0u) |
                                         (MODE != FORWARD ? 1u << 16 : 0u) | (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(BM >> 4) << 24);
        uint32_t stage = 0, phase = 0, acc = 0, accPhase = 0;
        bool ok = true;
        while (ok && walk.next(t)) {
            const int steps = walk.steps(t);
            if (steps == 0) continue;   // an expert without rows: the epilogue writes zeros
            if (!await(accEmpty + acc * 8, accPhase ^ 1, failed)) break;
            fenceAfter();
            const uint32_t d = tmem + acc * L::ACC;
            for (int k = 0; k < steps; ++k) {
                if (!await(full + stage * 8, phase, failed)) { ok = false; break; }
                fenceAfter();
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES;
                const int left = MODE == WEIGHTS ? t.end - t.begin - k * BK : p.sum - k * BK, parts = min(BK, left + 15) / 16;
                if (MODE == WEIGHTS && left < parts * 16) {
                    // the last rows of the step belong to another expert
                    const int rows = parts * 16 - left;
                    for (int i = lane; i < rows * ((BM + BN) / 64) * 8; i += 32) {
                        const int box = i / (rows * 8), r = left + i / 8 % rows, chunk = i % 8;
                        *reinterpret_cast<uint4*>(base + stage * L::STAGE + box * BOX + r * 128 + chunk * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fenceProxyAsync();
                    __syncwarp();
                }
                if (lane == 0) {
                    const uint64_t descA = operandDescriptor(a, MODE == WEIGHTS ? BOX : 16), descB = operandDescriptor(b, MODE == FORWARD ? 16 : BOX);
                    // 16 along the sum: 32 bytes of a K-major row, 16 rows of an MN-major block
                    for (int i = 0; i < parts; ++i)
                        mma(d, descA + i * (MODE == WEIGHTS ? 2048 >> 4 : 32 >> 4), descB + i * (MODE == FORWARD ? 32 >> 4 : 2048 >> 4), instruction, k + i > 0);
                    mmaCommit(empty + stage * 8);
                    if (k == steps - 1) mmaCommit(accFull + acc * 8);
                }
                __syncwarp();
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
            if (++acc == 2) { acc = 0; accPhase ^= 1; }
        }
    } else {
        // ---- epilogue --------------------------------------------------------------------------------------------------
        const int quarter = warp & 3;   // lanes of tensor memory this warp may read
        unsigned char* mine = outStage + (warp - 2) * 32 * 128;
        T* out = static_cast<T*>(p.out);
        uint32_t acc = 0, accPhase = 0;
        while (walk.next(t)) {
            const int steps = walk.steps(t);
            if (steps > 0) {
                if (!await(accFull + acc * 8, accPhase, failed)) break;
                fenceAfter();
            }
            const uint32_t from = tmem + acc * L::ACC + (static_cast<uint32_t>(quarter * 32) << 16);
            // rows of D in memory: expert by expert, channels out (weights); the tile's own rows (else)
            const int rowsLeft = (MODE == WEIGHTS ? p.sum - t.row : t.end - t.row) - quarter * 32;
            const long long firstRow = (MODE == WEIGHTS ? static_cast<long long>(t.expert) * p.sum : 0ll) + t.row + quarter * 32;
            const bool split = MODE == WEIGHTS && t.units > 1;
            float* partial = nullptr;
            if constexpr (MODE == WEIGHTS) {
                const long long item = before[t.expert] + t.unit, tileAt = static_cast<long long>(t.row / BM) * p.columnTiles + t.column / BN;
                partial = p.partial + ((item * p.rowTiles * p.columnTiles + tileAt) * BM + quarter * 32 + lane) * BN;
            }
            for (int c0 = 0; c0 < BN && t.column + c0 < p.columns; c0 += 64) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[32];
                    if (steps > 0) tmemLoad32(from + c0 + h * 32, v);
                    else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    }
                    if (MODE == WEIGHTS && split) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(partial + c0 + h * 32 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        continue;
                    }
                    if (MODE == FORWARD && p.bias != nullptr) {
                        const T* bias = static_cast<const T*>(p.bias) + static_cast<long long>(t.expert) * p.columns;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const int c = t.column + c0 + h * 32 + i;
                            v[i] += c < p.columns ? Element<T>::to(bias[c]) : 0.f;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float f[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) f[k] = v[i * 8 + k];
                        store<T, 8>(reinterpret_cast<T*>(mine + lane * 128 + (((h * 4 + i) ^ (lane & 7)) << 4)), pack<T, 8>(f));
                    }
                }
                if (MODE == WEIGHTS && split) continue;
                __syncwarp();
                if (p.wideStore) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int r = i * 4 + (lane >> 3), chunk = lane & 7, c = t.column + c0 + chunk * 8;
                        if (r < rowsLeft && c < p.columns)
                            store<T, 8>(out + (firstRow + r) * p.outStride + c, load<T, 8>(reinterpret_cast<const T*>(mine + r * 128 + ((chunk ^ (r & 7)) << 4))));
                    }
                } else {
                    for (int r = 0; r < 32 && r < rowsLeft; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int k = h * 32 + lane, c = t.column + c0 + k;
                            if (c < p.columns)
                                out[(firstRow + r) * p.outStride + c] = *reinterpret_cast<const T*>(mine + r * 128 + (((k >> 3) ^ (r & 7)) << 4) + (k & 7) * 2);
                        }
                }
                __syncwarp();
            }
            if (steps > 0) {
                fenceBefore();
                __syncwarp();
                if (lane == 0) barrierArrive(accEmpty + acc * 8);
                if (++acc == 2) { acc = 0; accPhase ^= 1; }
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
    }
    fenceBefore();
    __syncthreads();
    fenceAfter();
    if (warp == 1) {
        if (*failed != 0) {
            // products that were issued end before the tensor memory is given back
            if (lane == 0) {
                mmaCommit(drain);
                for (uint32_t n = 0; n < WAIT_LIMIT && !barrierTest(drain, 0); ++n) {}
                atomicOr(p.status, 1);
            }
            __syncwarp();
        }
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM) : "memory");
    }
}

// adds up the partial sums of the weight gradients of experts with more than one item: a block per 16 rows of a tile of an expert
template <class T, int BN>
__global__ void __launch_bounds__(256) expert_join_kernel(const __grid_constant__ ProductArgs p)
{
    const int tiles = p.rowTiles * p.columnTiles;
    const int expert = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const int before = p.plan[expert], units = p.plan[expert + 1] - before;
    if (units == 1) return;
    const long long unitStride = static_cast<long long>(tiles) * BM * BN;
    const float* from = p.partial + before * unitStride + static_cast<long long>(tile) * BM * BN;
    const int row0 = tile / p.columnTiles * BM, column0 = tile % p.columnTiles * BN;
    for (int i = threadIdx.x; i < 16 * BN; i += 256) {
        const int r = blockIdx.y * 16 + i / BN, c = i % BN;
        if (row0 + r >= p.sum || column0 + c >= p.columns) continue;
        float sum = 0.f;
#pragma unroll 4
        for (int u = 0; u < units; ++u) sum += from[u * unitStride + r * BN + c];
        static_cast<T*>(p.out)[(static_cast<long long>(expert) * p.sum + row0 + r) * p.outStride + column0 + c] = Element<T>::from(sum);
    }
}

// ---- bias gradient: column sums of an expert's rows ------------------------------------------------------------------------
// blockIdx.x: expert, blockIdx.y: 32 x 8 columns. 8 warps take strided rows, then join.
template <class T>
__global__ void __launch_bounds__(256) expert_bias_kernel(const __grid_constant__ ProductArgs p, const T* __restrict__ dy, long long stride, T* __restrict__ out)
{
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
// rows of `columns` elements -> rows of `padded` (a multiple of 8) elements, zeros behind
template <class T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T* __restrict__ in, long long stride, T* __restrict__ out, long long rows, int columns, int padded)
{
    const long long total = rows * padded;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += static_cast<long long>(gridDim.x) * 256) {
        const long long r = i / padded;
        const int c = static_cast<int>(i - r * padded);
        out[i] = c < columns ? in[r * stride + c] : Element<T>::from(0.f);
    }
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
    const CUresult r = encode(&map, type == TYPE_HALF ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, matrices > 0 ? 3 : 2, const_cast<void*>(data),
                              dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }
int pad8(int n) { return (n + 7) / 8 * 8; }
// rows the TMA can read where they lie
bool direct(const void* data, long long stride, int columns) { return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && stride % 8 == 0 && stride >= columns; }

int tileWidth(int columns) { return columns <= 64 ? 64 : columns <= 128 ? 128 : 256; }

// rows per item of the weight gradient: enough items that every SM gets a few
int weightChunk(const ExpertArgs& a, int tiles)
{
    const long long items = std::max<long long>(1, 4ll * a.numSMs / tiles);
    return static_cast<int>(std::min<long long>(std::max<long long>((a.rows / items + 63) / 64 * 64, 512), 1ll << 30));
}

// scratch: [x | weight | dy in a form the TMA reads, where needed | partial sums of the weight gradients]
struct Scratch {
    size_t x, weight, gradY, partial, plan, bytes;
    int chunk, rowTiles, columnTiles, width;
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
        width = tileWidth(a.channelsIn);
        rowTiles = (a.channelsOut + BM - 1) / BM;
        columnTiles = (a.channelsIn + width - 1) / width;
        const int tiles = rowTiles * columnTiles;
        chunk = weightChunk(a, tiles);
        const size_t items = a.rows > chunk ? a.experts + rows / chunk : 0;
        partial = take(weights && items > 0, items * tiles * BM * width * 4);
        plan = take(weights && items > 0, (static_cast<size_t>(a.experts) + 1) * 4);
    }
};

template <class T>
cudaError_t readable(const void*& data, long long& stride, long long rows, int columns, void* scratch, int numSMs, cudaStream_t stream)
{
    if (direct(data, stride, columns)) return cudaSuccess;
    const int padded = pad8(columns);
    const long long blocks = std::min<long long>((rows * padded + 255) / 256, numSMs * 16ll);
    pad_rows_kernel<T><<<static_cast<unsigned>(std::max(1ll, blocks)), 256, 0, stream>>>(static_cast<const T*>(data), stride, static_cast<T*>(scratch), rows, columns, padded);
    data = scratch;
    stride = padded;
    return cudaGetLastError();
}

template <class T, int MODE, int BN>
cudaError_t launchProduct(const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& p, int blocks, cudaStream_t stream)
{
    auto* kernel = expert_product_kernel<T, MODE, BN>;
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), Layout<BN>::bytes(EXPERTS_MAX));
    if (e != cudaSuccess) return e;
    kernel<<<blocks, BLOCK, Layout<BN>::bytes(p.experts), stream>>>(a, b, p);
    return cudaGetLastError();
}
template <class T, int MODE>
cudaError_t launchWidth(const CUtensorMap& a, const CUtensorMap& b, const ProductArgs& p, int blocks, cudaStream_t stream)
{
    switch (tileWidth(p.columns)) {
    case 64: return launchProduct<T, MODE, 64>(a, b, p, blocks, stream);
    case 128: return launchProduct<T, MODE, 128>(a, b, p, blocks, stream);
    default: return launchProduct<T, MODE, 256>(a, b, p, blocks, stream);
    }
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

template <class T>
cudaError_t forward(const ExpertArgs& a, cudaStream_t stream)
{
    const Scratch s(a, false);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    const void *x = a.x.data, *w = a.weight;
    long long xStride = a.x.stride, wStride = a.channelsIn;
    cudaError_t e = readable<T>(x, xStride, a.rows, a.channelsIn, base + s.x, a.numSMs, stream);
    if (e == cudaSuccess) e = readable<T>(w, wStride, static_cast<long long>(a.experts) * a.channelsOut, a.channelsIn, base + s.weight, a.numSMs, stream);
    CUtensorMap mapX, mapW;
    if (e == cudaSuccess) e = encodeMap(mapX, a.type, x, 0, a.rows, a.channelsIn, xStride);
    if (e == cudaSuccess) e = encodeMap(mapW, a.type, w, a.experts, a.channelsOut, a.channelsIn, wStride);
    if (e != cudaSuccess) return e;
    ProductArgs p = common(a);
    p.columns = a.channelsOut;
    p.sum = a.channelsIn;
    p.columnTiles = (p.columns + tileWidth(p.columns) - 1) / tileWidth(p.columns);
    p.out = a.y.data;
    p.outStride = a.y.stride;
    p.bias = a.bias;
    p.wideStore = wideOut(p.out, p.outStride, p.columns);
    return launchWidth<T, FORWARD>(mapX, mapW, p, a.numSMs, stream);
}

template <class T>
cudaError_t adjoint(const ExpertArgs& a, cudaStream_t stream)
{
    const Scratch s(a, true);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    cudaError_t e = cudaSuccess;
    if (a.gradBias != nullptr) {
        ProductArgs p = common(a);
        p.columns = a.channelsOut;
        expert_bias_kernel<T><<<dim3(a.experts, (a.channelsOut + 31) / 32), 256, 0, stream>>>(p, static_cast<const T*>(a.gradY.data), a.gradY.stride, static_cast<T*>(a.gradBias));
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
    if (e == cudaSuccess) e = readable<T>(dy, dyStride, a.rows, a.channelsOut, base + s.gradY, a.numSMs, stream);
    if (e == cudaSuccess) e = encodeMap(mapY, a.type, dy, 0, a.rows, a.channelsOut, dyStride);
    if (e == cudaSuccess && a.gradX.data != nullptr) {
        e = readable<T>(w, wStride, static_cast<long long>(a.experts) * a.channelsOut, a.channelsIn, base + s.weight, a.numSMs, stream);
        if (e == cudaSuccess) e = encodeMap(mapW, a.type, w, a.experts, a.channelsOut, a.channelsIn, wStride);
        if (e != cudaSuccess) return e;
        ProductArgs p = common(a);
        p.columns = a.channelsIn;
        p.sum = a.channelsOut;
        p.columnTiles = (p.columns + tileWidth(p.columns) - 1) / tileWidth(p.columns);
        p.out = a.gradX.data;
        p.outStride = a.gradX.stride;
        p.wideStore = wideOut(p.out, p.outStride, p.columns);
        e = launchWidth<T, INPUT>(mapY, mapW, p, a.numSMs, stream);
    }
    if (e == cudaSuccess && a.gradWeight != nullptr) {
        e = readable<T>(x, xStride, a.rows, a.channelsIn, base + s.x, a.numSMs, stream);
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
        p.plan = a.rows > s.chunk ? reinterpret_cast<int*>(base + s.plan) : nullptr;
        p.wideStore = wideOut(p.out, p.outStride, p.columns);
        e = launchWidth<T, WEIGHTS>(mapY, mapX, p, a.numSMs, stream);
        if (e == cudaSuccess && a.rows > s.chunk) {
            const dim3 grid(a.experts * s.rowTiles * s.columnTiles, BM / 16);
            if (s.width == 64) expert_join_kernel<T, 64><<<grid, 256, 0, stream>>>(p);
            else if (s.width == 128) expert_join_kernel<T, 128><<<grid, 256, 0, stream>>>(p);
            else expert_join_kernel<T, 256><<<grid, 256, 0, stream>>>(p);
            e = cudaGetLastError();
        }
    }
    return e;
}

} // namespace

size_t expertBytes(const ExpertArgs& a, bool adjoint) { return a.rows == 0 ? 0 : Scratch(a, adjoint).bytes; }

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
