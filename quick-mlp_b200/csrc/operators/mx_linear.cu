// Products of feature rows with microscaled 4-bit matrices, one matrix per expert: rows [offsets[e], offsets[e + 1]) of x belong to expert e.
//
//   y_r = W_e q(x_r) + b_e          W_e: (channels out, channels in) in 4 bits; q: the row in 4 bits (mx.cuh)
//   dx_r = W_e^T dy_r               (straight through q), W_e decoded to 16 bits, which is exact, and the product of expert_linear.cu
//
// Two kernels. The first quantises the rows, tile by tile of 128 rows of one expert, so that a tile's scales lie as the tensor core wants them. The second
// is the product D (128 x BN, fp32 in tensor memory) += A B, 256 channels in a step: codes by TMA in boxes of 64 rows x 128 bytes (256 channels), 128-byte
// swizzled, both operands K-major; scales by TMA in tiles of 512 bytes, copied to tensor memory by tcgen05.cp in front of the products that use them. A
// product multiplies 64 channels, blocks of 32 with their two scales (kind::mxf4), exactly, and adds them up in fp32. What lies outside a matrix arrives as zeros.
// A tile that reaches behind its expert's last row reads rows of the next one, which only fill rows of D that are not stored.
//
// One persistent block per SM, or a pair of blocks that share tiles of 256 x 256: a TMA warp, an MMA warp, two groups of four epilogue warps,
// one per accumulator. Tensor memory has no room for two accumulators of 256 columns and the scales: there the second begins 64 columns before
// the first one's end, and the epilogue reads the shared columns first.
// Waits are bounded: on a timeout the block drains, gives its tensor memory back and sets the library's status word.
#include "mx.cuh"
#include "products.cuh"

#include <algorithm>

namespace qmlp {
namespace kernel {
namespace {

using namespace mx;
using namespace products;

constexpr int STEP_CHANNELS = 256, SCALE_BYTES = 2 * MX_TILE_BYTES;   // channels of a step (128 bytes of codes), scales of 128 rows of a step

// BN: columns of D; CTAS: blocks that share a tile, each with BM rows of D and BN / CTAS of the columns of B
template <int BN, int CTAS>
struct MxLayout {
    static constexpr int BCOLS = BN / CTAS, ABYTES = BM * 128, BBYTES = BCOLS * 128;
    static constexpr int BTILES = (BN + MX_TILE - 1) / MX_TILE;       // tiles of scales of the columns (each block has all of them)
    static constexpr int SCALES = ABYTES + BBYTES, STAGE = SCALES + SCALE_BYTES * (1 + BTILES);
    static constexpr int STAGES = std::min(8, 192 * 1024 / STAGE);
    // tensor memory: accumulators, then two sets of scales, used in turn: of 128 rows (4 columns) for two times 128 channels, of the columns likewise
    static constexpr bool OVERLAP = BN == 256;
    static constexpr int SECOND = OVERLAP ? BN - 64 : BN;             // column of the second accumulator
    static constexpr int SCALE_AT = SECOND + BN, SCALE_SET = 32, SCALE_B = 8, SCALE_B_STEP = 4 * BTILES;
    static constexpr int TMEM = SCALE_AT + 2 * SCALE_SET <= 256 ? 256 : 512;
    static constexpr int EPILOGUE = 32 * 64 + BN * 4, OUT = EPILOGUE_WARPS * EPILOGUE;   // per warp: 32 rows x 32 elements of 16 bits, a bias
    // barriers: full, empty (STAGES each), accumulator full, empty, overlap free (2 each), drain; then flag and tensor memory
    static constexpr int FULL = 0, EMPTY = 64, ACC_FULL = 128, ACC_EMPTY = 144, SHARED_FREE = 160, DRAIN = 176, FAILED = 184, BASE = 188, BARS = 192;
    // 1 KB for the alignment of the ring
    static constexpr int bytes(int experts) { return 1024 + STAGES * STAGE + OUT + BARS + listInts(experts) * 4; }
    static_assert(SCALE_AT + 2 * SCALE_SET <= TMEM && SCALE_B + 2 * SCALE_B_STEP <= SCALE_SET, "tensor memory");
    static_assert(STAGE % 1024 == 0 && STAGES >= 3, "ring");
    static_assert(bytes(EXPERTS_MAX) + 512 <= 227 * 1024, "shared memory");
};
constexpr int MX_THREADS = (2 + EPILOGUE_WARPS) * 32;

// ---- PTX ---------------------------------------------------------------------------------------------------------------
// a product of 64 channels; the instruction descriptor names the scales' places within their words
template <int CTAS>
__device__ __forceinline__ void mmaMx(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t scaleA, uint32_t scaleB, uint32_t accumulate)
{
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
                     "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
                     "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(scaleA), "r"(scaleB), "r"(accumulate), "r"(lead) : "memory");
}
// 512 bytes of shared memory (of both blocks, each its own) to 4 columns of tensor memory, 16 bytes a lane, the same in all four quarters
template <int CTAS>
__device__ __forceinline__ void copyScales(uint32_t lead, uint32_t to, uint64_t from)
{
    if constexpr (CTAS == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(to), "l"(from), "r"(lead) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(to), "l"(from), "r"(lead) : "memory");
}
// descriptor of a tile of scales: no swizzle, groups of 8 rows of 16 bytes lie 128 bytes apart
__device__ __forceinline__ uint64_t scaleDescriptor(uint32_t address) { return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (8ull << 32) | (1ull << 46); }

// ---- the rows in 4 bits ----------------------------------------------------------------------------------------------------
// Tiles of 128 rows of one expert, in the order of the product's units (of tileRows rows): tile t of all is part t % (tileRows / 128) of unit t / (tileRows / 128).
template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_rows_kernel(const __grid_constant__ ProductArgs p, const T* __restrict__ x, long long stride, unsigned char* __restrict__ codes,
                                                               unsigned char* __restrict__ scales, int chunks, int codeBytes)
{
    extern __shared__ int lists[];
    __shared__ uint4 words[2][MX_TILE / 4];
    chained();
    int *bounds = lists, *before = lists + listStride(p.experts);
    planExperts<FORWARD>(p, bounds, before, nullptr, TILE_THREADS);
    __syncthreads();
    const int parts = p.tileRows / MX_TILE;
    const long long items = static_cast<long long>(before[p.experts]) * parts * chunks;
    int flip = 0;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const long long tile = item / chunks;
        const int chunk = static_cast<int>(item - tile * chunks), unit = static_cast<int>(tile / parts), part = static_cast<int>(tile - static_cast<long long>(unit) * parts);
        int low = 0, high = p.experts;   // the last expert whose units begin at or before this one (experts without units end up in front of it)
        while (high - low > 1) {
            const int middle = (low + high) / 2;
            if (before[middle] <= unit) low = middle;
            else high = middle;
        }
        const long long begin = bounds[low] + static_cast<long long>(unit - before[low]) * p.tileRows + part * MX_TILE;
        const long long left = bounds[low + 1] - begin;
        if (left <= 0) continue;   // the second half of a unit's rows may be empty
        quantizeTile<T, LANES, ALIGNED>(x + begin * stride, stride, static_cast<int>(min(left, static_cast<long long>(MX_TILE))), chunk, p.sum, codes + begin * codeBytes, codeBytes,
                                        scales + item * MX_TILE_BYTES, reinterpret_cast<uint32_t*>(words[flip]));
        flip ^= 1;   // (the next barrier lies between this use and the next of the same words)
    }
}

// ---- the product -------------------------------------------------------------------------------------------------------------
template <class T, int BN, int CTAS>
__global__ void __launch_bounds__(MX_THREADS, 1)
    mx_product_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapScaleA,
                      const __grid_constant__ CUtensorMap mapScaleB, const __grid_constant__ ProductArgs p, int chunks)
{
    using L = MxLayout<BN, CTAS>;
    extern __shared__ unsigned char dynamic[];
    const uint32_t raw = smemAddress(dynamic), ring = (raw + 1023u) & ~1023u;
    unsigned char* base = dynamic + (ring - raw);
    unsigned char* outStage = base + L::STAGES * L::STAGE;
    const uint32_t bars = ring + L::STAGES * L::STAGE + L::OUT;
    const uint32_t full = bars + L::FULL, empty = bars + L::EMPTY, accFull = bars + L::ACC_FULL, accEmpty = bars + L::ACC_EMPTY, sharedFree = bars + L::SHARED_FREE;
    volatile int* failed = reinterpret_cast<volatile int*>(outStage + L::OUT + L::FAILED);
    uint32_t* tmemBase = reinterpret_cast<uint32_t*>(outStage + L::OUT + L::BASE);
    int *bounds = reinterpret_cast<int*>(outStage + L::OUT + L::BARS), *before = bounds + listStride(p.experts);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 1 ? 0u : clusterRank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            barrierInit(full + s * 8, CTAS);
            barrierInit(empty + s * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            barrierInit(accFull + i * 8, 1);
            barrierInit(accEmpty + i * 8, 4 * CTAS);
            barrierInit(sharedFree + i * 8, 4 * CTAS);
        }
        barrierInit(bars + L::DRAIN, 1);
        *failed = 0;
        barrierInitDone();
    }
    if (warp == 1) tmemAlloc<CTAS>(smemAddress(tmemBase), L::TMEM);
    chained();
    planExperts<FORWARD>(p, bounds, before, nullptr, MX_THREADS);
    fenceBefore();
    __syncthreads();
    if constexpr (CTAS > 1) clusterSync();   // the other block's barriers are set
    fenceAfter();
    const uint32_t tmem = *tmemBase;
    const int steps = (p.sum + STEP_CHANNELS - 1) / STEP_CHANNELS;
    Walk<FORWARD, BN, CTAS> walk(p, bounds, before, nullptr, 0, 1);
    Tile t;
    InFlight copies;   // of warp 0

    if (warp == 0) {
        // ---- operands -------------------------------------------------------------------------------------------------
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0;
        long long issued = 0;
        bool ok = true;
        const int columnScaleTiles = (p.columns + MX_TILE - 1) / MX_TILE;
        while (ok && walk.next(t)) {
            if (__all_sync(0xffffffffu, t.expert < 0)) continue;   // no tile for this block in the last round
            const int row = t.row + rank * BM, column = t.column + rank * L::BCOLS;
            const int boxesA = boxes(t.end - row, BM / 64), boxesB = boxes(p.columns - column, L::BCOLS / 64);
            const uint32_t bytes = (boxesA + boxesB) * BOX + SCALE_BYTES * (1 + L::BTILES);   // of this block; of both blocks:
            const uint32_t allBytes = CTAS == 1 ? bytes : bytes + (boxes(t.end - row - BM, BM / 64) + boxes(p.columns - column - L::BCOLS, L::BCOLS / 64)) * BOX + SCALE_BYTES * (1 + L::BTILES);
            // tiles of scales, each a row of the scales' maps (the expert's tiles of 128 columns: one behind the last is the next expert's, or zeros)
            const int scaleA = (t.slot * CTAS + static_cast<int>(rank)) * chunks, scaleB = (t.expert * columnScaleTiles + t.column / MX_TILE) * chunks;
            for (int k = 0; __all_sync(0xffffffffu, k < steps); ++k) {
                if (!await(empty + stage * 8, phase ^ 1, failed)) { ok = false; break; }
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES, s = a + L::SCALES;
                const uint32_t ready = CTAS == 1 ? full + stage * 8 : inBlock(full + stage * 8, 0);
                if (lead && rank == 0) {
                    // the leader expects the bytes of both blocks, and arrives for both
                    barrierExpect(full + stage * 8, allBytes);
                    if (CTAS > 1) barrierArrive(full + stage * 8);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < BM / 64; ++i) tmaLoad2<CTAS>(lead && i < boxesA, a + i * BOX, &mapA, k * 32, row + i * 64, ready);
#pragma unroll
                for (int i = 0; i < L::BCOLS / 64; ++i) tmaLoad3<CTAS>(lead && i < boxesB, b + i * BOX, &mapB, k * 32, column + i * 64, t.expert, ready);
                tmaLoad2<CTAS>(lead, s, &mapScaleA, 0, scaleA + k * 2, ready);
#pragma unroll
                for (int i = 0; i < L::BTILES; ++i) tmaLoad2<CTAS>(lead, s + SCALE_BYTES * (1 + i), &mapScaleB, 0, scaleB + i * chunks + k * 2, ready);
                ++issued;
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
        }
        copies.stage = stage;
        copies.phase = phase;
        copies.count = rank == 0 ? static_cast<int>(min(issued, static_cast<long long>(L::STAGES))) : 0;   // (the other block's arrive here too)
    } else if (warp == 1) {
        // ---- products -------------------------------------------------------------------------------------------------
        // e2m1 operands, power-of-two scales
        constexpr uint32_t instruction = (1u << 7) | (1u << 10) | (static_cast<uint32_t>(BN >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>((BM * CTAS) >> 7) << 27);
        const uint32_t lead = electOne();
        uint32_t stage = 0, phase = 0, acc = 1, accPhases = 0;   // accPhases: one bit per accumulator
        uint32_t set = 0, before1 = 0, before2 = 0;              // set of scales; barrier and parity (bit 31) of the step before, of the one before that
        bool ok = rank == 0;
        while (ok && walk.next(t)) {
            acc ^= 1;                   // the tiles' numbers alternate between the accumulators
            if (__all_sync(0xffffffffu, t.expert < 0)) continue;   // no tile for this block in the last round
            if (!await(accEmpty + acc * 8, (accPhases >> acc & 1) ^ 1, failed)) break;
            if constexpr (L::OVERLAP)
                if (!await(sharedFree + (acc ^ 1) * 8, (accPhases >> (acc ^ 1) & 1) ^ 1, failed)) break;
            accPhases ^= 1u << acc;
            fenceAfter();
            const uint32_t d = tmem + acc * L::SECOND;
            for (int k = 0; __all_sync(0xffffffffu, k < steps); ++k) {
                if (!await(full + stage * 8, phase, failed)) { ok = false; break; }
                // the products that read this set of scales are done (those of the step before keep the tensor core busy meanwhile)
                if (before2 != 0 && !await(before2 & 0x7fffffffu, before2 >> 31, failed)) { ok = false; break; }
                fenceAfter();
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES, s = a + L::SCALES, scales = tmem + L::SCALE_AT + set * L::SCALE_SET;
                const int parts = min(STEP_CHANNELS, p.sum - k * STEP_CHANNELS + 63) / 64;
                const uint64_t descA = operandDescriptor(a, 16), descB = operandDescriptor(b, 16), descS = scaleDescriptor(s);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    copyScales<CTAS>(lead && parts > 2 * c, scales + c * 4, descS + c * (MX_TILE_BYTES >> 4));
#pragma unroll
                    for (int i = 0; i < L::BTILES; ++i)
                        copyScales<CTAS>(lead && parts > 2 * c, scales + L::SCALE_B + c * L::SCALE_B_STEP + i * 4, descS + ((SCALE_BYTES * (1 + i) + c * MX_TILE_BYTES) >> 4));
                }
                // 64 channels: 32 bytes of a row, two scales of a word of four
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mmaMx<CTAS>(lead && i < parts, d, descA + i * (32 >> 4), descB + i * (32 >> 4), instruction | (i & 1 ? (2u << 29) | (2u << 4) : 0u), scales + i / 2 * 4,
                                scales + L::SCALE_B + i / 2 * L::SCALE_B_STEP, i > 0 ? 1u : k > 0 ? 1u : 0u);
                mmaCommit<CTAS>(lead, empty + stage * 8);
                mmaCommit<CTAS>(lead && k == steps - 1, accFull + acc * 8);
                before2 = before1;
                before1 = (empty + stage * 8) | phase << 31;
                set ^= 1;
                if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
            }
        }
    } else {
        // ---- epilogue: two groups of four warps, one per accumulator -------------------------------------------------------
        const int group = (warp - 2) / 4, quarter = warp & 3;   // quarter: lanes of tensor memory this warp may read
        unsigned char* mine = outStage + (warp - 2) * L::EPILOGUE;
        float* mineBias = reinterpret_cast<float*>(mine + 32 * 64);
        const uint32_t released = CTAS == 1 ? accEmpty + group * 8 : inBlock(accEmpty + group * 8, 0);
        const uint32_t sharedReleased = CTAS == 1 ? sharedFree + group * 8 : inBlock(sharedFree + group * 8, 0);
        auto release = [&](uint32_t bar) {
            fenceBefore();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CTAS == 1) barrierArrive(bar);
                else clusterArriveBarrier(bar);
            }
        };
        T* out = static_cast<T*>(p.out);
        uint32_t accPhase = 0;
        walk = Walk<FORWARD, BN, CTAS>(p, bounds, before, nullptr, group, EPILOGUE_GROUPS);
        while (walk.next(t)) {
            if (t.expert < 0) break;
            const int tileRow = t.row + rank * BM;
            if (p.bias != nullptr) {
                const T* row = static_cast<const T*>(p.bias) + static_cast<long long>(t.expert) * p.columns + t.column;
#pragma unroll
                for (int i = lane; i < BN; i += 32) mineBias[i] = t.column + i < p.columns ? Element<T>::to(row[i]) : 0.f;
                __syncwarp();
            }
            if (!await(accFull + group * 8, accPhase, failed)) break;
            accPhase ^= 1;
            fenceAfter();
            const uint32_t from = tmem + group * L::SECOND + (static_cast<uint32_t>(quarter * 32) << 16);
            const int rowsLeft = t.end - tileRow - quarter * 32;
            const long long firstRow = tileRow + quarter * 32;
            // 64 columns of the accumulator at a time, 32 through shared memory; the columns that the accumulators share first: the last of one, the
            // first of the other
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) {
                const int pair = L::OVERLAP && group == 0 ? (i + BN / 64 - 1) % (BN / 64) : i;
                const bool used = t.column + pair * 64 < p.columns && rowsLeft > 0;
                float v[2][32];
                if (used) {
                    tmemLoad32(from + pair * 64, v[0]);
                    tmemLoad32(from + pair * 64 + 32, v[1]);
                    tmemWait(v[0], v[1]);
                }
                if (L::OVERLAP && i == 0) release(sharedReleased);
                if (!used) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c0 = pair * 64 + h * 32;
                    if (t.column + c0 >= p.columns) break;
                    if (p.bias != nullptr) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(mineBias + c0 + j);
                            v[h][j] += f.x;
                            v[h][j + 1] += f.y;
                            v[h][j + 2] += f.z;
                            v[h][j + 3] += f.w;
                        }
                    }
                    storeTile<T>(v[h], mine, out + firstRow * p.outStride + t.column, p.outStride, rowsLeft, c0, p.columns - t.column, p.wideStore);
                }
            }
            release(released);
        }
        // rows before the first and behind the last expert belong to nobody
        const int first = bounds[0], last = bounds[p.experts];
        const long long warps = static_cast<long long>(gridDim.x) * EPILOGUE_WARPS, me = static_cast<long long>(blockIdx.x) * EPILOGUE_WARPS + (warp - 2);
        for (long long r = me; r < first + (p.rows - last); r += warps) {
            T* row = out + (r < first ? r : last + (r - first)) * p.outStride;
            for (int c = lane; c < p.columns; c += 32) row[c] = Element<T>::from(0.f);
        }
    }
    fenceBefore();
    __syncthreads();
    fenceAfter();
    if (*failed != 0 && warp == 0) {
        copies.land(full, L::STAGES);
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

// ---- host ------------------------------------------------------------------------------------------------------------------
// `matrices` matrices of `rows` rows of `bytes` bytes, one behind the other (0: one, for a 2-D map), boxes of boxRows x boxBytes
cudaError_t encodeBytes(CUtensorMap& map, const void* data, long long matrices, long long rows, int bytes, int boxBytes, int boxRows, bool swizzle)
{
    const EncodeFn encode = encoder();
    if (encode == nullptr) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(bytes / 4), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(matrices)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(bytes) * rows};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(boxBytes / 4), static_cast<cuuint32_t>(boxRows), 1}, one[3] = {1, 1, 1};
    auto run = [&] {
        return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, matrices > 0 ? 3 : 2, const_cast<void*>(data), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = run();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {   // a thread's first call: the driver wants a context, which the runtime binds
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaSetDevice(device);
        if (e != cudaSuccess) return e;
        r = run();
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

struct Shape {
    int width, ctas;
};
Shape shapeOf(const MxLinearArgs& a)
{
    const int columns = static_cast<int>(a.weight.rows);
    if (columns <= 64) return {64, 1};
    if (columns <= 128 || a.rows / a.weight.matrices < 512) return {128, 1};
    return {256, 2};
}
// tiles of 128 rows, none with rows of two experts, a multiple of ctas per expert: an upper bound
long long rowTiles(const MxLinearArgs& a, int ctas)
{
    return (a.rows / (MX_TILE * ctas) + std::min<long long>(a.rows, a.weight.matrices)) * ctas;
}
struct MxScratch {
    size_t scales, bytes;   // codes lie at the start
    MxScratch(const MxLinearArgs& a)
    {
        scales = align256(static_cast<size_t>(a.rows) * mxCodeBytes(a.weight.channels));
        bytes = scales + align256(static_cast<size_t>(rowTiles(a, shapeOf(a).ctas)) * mxTiles(a.weight.channels) * MX_TILE_BYTES);
    }
};

template <class T, int LANES, bool ALIGNED>
cudaError_t launchRows(const MxLinearArgs& a, const ProductArgs& p, unsigned char* codes, unsigned char* scales, cudaStream_t stream)
{
    auto* kernel = mx_rows_kernel<T, LANES, ALIGNED>;
    const long long items = rowTiles(a, p.tileRows / MX_TILE) * mxTiles(p.sum);
    launchChained(kernel, static_cast<unsigned>(std::min<long long>(items, a.numSMs * 6)), TILE_THREADS, 2 * listStride(p.experts) * sizeof(int), stream, 1, p,
                  static_cast<const T*>(a.x.data), a.x.stride, codes, scales, mxTiles(p.sum), mxCodeBytes(p.sum));
    return cudaGetLastError();
}
template <class T>
cudaError_t quantizeRows(const MxLinearArgs& a, const ProductArgs& p, unsigned char* codes, unsigned char* scales, cudaStream_t stream)
{
    const bool aligned = (reinterpret_cast<uintptr_t>(a.x.data) & 15) == 0 && a.x.stride % 8 == 0 && p.sum % 8 == 0;
    switch (lanesOf(p.sum)) {
    case 4: return aligned ? launchRows<T, 4, true>(a, p, codes, scales, stream) : launchRows<T, 4, false>(a, p, codes, scales, stream);
    case 8: return aligned ? launchRows<T, 8, true>(a, p, codes, scales, stream) : launchRows<T, 8, false>(a, p, codes, scales, stream);
    default: return aligned ? launchRows<T, 16, true>(a, p, codes, scales, stream) : launchRows<T, 16, false>(a, p, codes, scales, stream);
    }
}

template <class T, int BN, int CTAS>
cudaError_t launchMx(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& sa, const CUtensorMap& sb, const ProductArgs& p, int numSMs, cudaStream_t stream)
{
    auto* kernel = mx_product_kernel<T, BN, CTAS>;
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), MxLayout<BN, CTAS>::bytes(EXPERTS_MAX));
    if (e != cudaSuccess) return e;
    return launchChained(kernel, numSMs / CTAS * CTAS, MX_THREADS, MxLayout<BN, CTAS>::bytes(p.experts), stream, CTAS, a, b, sa, sb, p, mxTiles(p.sum));
}

template <class T>
cudaError_t forward(const MxLinearArgs& a, cudaStream_t stream)
{
    const Shape shape = shapeOf(a);
    const MxScratch s(a);
    unsigned char *codes = static_cast<unsigned char*>(a.scratch), *scales = codes + s.scales;
    ProductArgs p{};
    p.rows = a.rows;
    p.experts = static_cast<int>(a.weight.matrices);
    p.columns = static_cast<int>(a.weight.rows);
    p.sum = a.weight.channels;
    p.columnTiles = (p.columns + shape.width - 1) / shape.width;
    p.tileRows = BM * shape.ctas;
    p.offsets = a.offsets;
    p.out = a.y.data;
    p.outStride = a.y.stride;
    p.bias = a.bias;
    p.status = a.status;
    p.wideStore = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.outStride % 8 == 0 && p.columns % 8 == 0;
    const int chunks = mxTiles(p.sum), codeBytes = mxCodeBytes(p.sum);
    CUtensorMap mapA, mapB, mapScaleA, mapScaleB;
    cudaError_t e = encodeBytes(mapA, codes, 0, a.rows, codeBytes, 128, 64, true);
    if (e == cudaSuccess) e = encodeBytes(mapB, a.weight.codes, a.weight.matrices, p.columns, codeBytes, 128, 64, true);
    if (e == cudaSuccess) e = encodeBytes(mapScaleA, scales, 0, rowTiles(a, shape.ctas) * chunks, MX_TILE_BYTES, MX_TILE_BYTES, 2, false);
    if (e == cudaSuccess) e = encodeBytes(mapScaleB, a.weight.scales, 0, a.weight.matrices * mxTiles(p.columns) * chunks, MX_TILE_BYTES, MX_TILE_BYTES, 2, false);
    if (e == cudaSuccess) e = quantizeRows<T>(a, p, codes, scales, stream);
    if (e != cudaSuccess) return e;
    if (shape.width == 64) return launchMx<T, 64, 1>(mapA, mapB, mapScaleA, mapScaleB, p, a.numSMs, stream);
    if (shape.width == 128) return launchMx<T, 128, 1>(mapA, mapB, mapScaleA, mapScaleB, p, a.numSMs, stream);
    return launchMx<T, 256, 2>(mapA, mapB, mapScaleA, mapScaleB, p, a.numSMs, stream);
}

// the matrices in 16 bits, then the input gradient's and the bias gradient's scratch
size_t decodedBytes(const MxLinearArgs& a)
{
    return a.gradX.data == nullptr || a.rows == 0 ? 0 : align256(static_cast<size_t>(a.weight.matrices) * a.weight.rows * a.weight.channels * 2);
}
ExpertArgs decoded(const MxLinearArgs& a)
{
    ExpertArgs r{};
    r.rows = a.rows;
    r.experts = static_cast<int>(a.weight.matrices);
    r.channelsIn = a.weight.channels;
    r.channelsOut = static_cast<int>(a.weight.rows);
    r.type = a.type;
    r.numSMs = a.numSMs;
    r.weight = a.scratch;
    r.offsets = a.offsets;
    r.gradY = a.gradY;
    r.gradX = a.gradX;
    r.gradBias = a.gradBias;
    r.status = a.status;
    return r;
}

} // namespace

size_t mxLinearBytes(const MxLinearArgs& a) { return a.rows == 0 ? 0 : MxScratch(a).bytes; }
size_t mxLinearAdjointBytes(const MxLinearArgs& a) { return decodedBytes(a) + expertBytes(decoded(a), true); }

cudaError_t launchMxLinear(const MxLinearArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return a.type == TYPE_HALF ? forward<__half>(a, stream) : forward<__nv_bfloat16>(a, stream);
}
cudaError_t launchMxLinearAdjoint(const MxLinearArgs& a, cudaStream_t stream)
{
    ExpertArgs r = decoded(a);
    r.scratch = static_cast<unsigned char*>(a.scratch) + decodedBytes(a);
    if (decodedBytes(a) > 0) {
        const cudaError_t e = launchMxDequantize(a.weight, a.type, {a.scratch, a.weight.channels}, stream);
        if (e != cudaSuccess) return e;
    }
    return launchExpertAdjoint(r, stream);
}

} // namespace kernel
} // namespace qmlp
