// Products of feature rows with microscaled 4-bit matrices, one matrix per expert: rows [offsets[e], offsets[e + 1]) of x belong to expert e.
//
//   y_r = W_e q(x_r) + b_e          W_e: (channels out, channels in) in 4 bits; q: the row in 4 bits (mx.cuh)
//   dx_r = W_e^T dy_r               (straight through q), W_e decoded to 16 bits and the product of expert_linear.cu. bfloat16 holds every 4-bit number; half holds
//                                   27 neighbouring powers of two, so that W_e goes there divided by one where it leaves half's own (see mx_apart_kernel)
//
// Two kernels (one for small calls, and another for a few rows; the rules stand at the end). The first quantises the rows, tile by tile of 128 rows of one expert,
// so that a tile's scales lie as the tensor core wants them. The second is the product D (128 x BN, fp32 in tensor memory) += A B, 256 channels in a step: codes by TMA in boxes of 64 rows x 128 bytes (256 channels), 128-byte
// swizzled, both operands K-major; scales by TMA in tiles of 512 bytes, copied to tensor memory by tcgen05.cp in front of the products that use them. A
// product multiplies 64 channels, blocks of 32 with their two scales (kind::mxf4), exactly, and adds them up in fp32. What lies outside a matrix arrives as zeros.
// A tile that reaches behind its expert's last row reads rows of the next one, which only fill rows of D that are not stored.
//
// One persistent block per SM, or a pair of blocks that share tiles of 256 x 256: a TMA warp, an MMA warp, two groups of four epilogue warps,
// one per accumulator. Tensor memory has no room for two accumulators of 256 columns and the scales: there the second begins 64 columns before
// the first one's end, and the epilogue reads the shared columns first. 16384 rows of 4096 -> 4096 bfloat16: 31 us and 93 us (5.9 PFLOP/s); 16 experts, 131072 rows,
// 1024 -> 1024: 55 and 76 us, of which the shared columns cost about a third (a tile's 4 steps take 2050 clocks, until the next one's first product goes out 1200 more pass:
// accumulator complete, 64 columns read, released, issued). All eight warps of the epilogue on every tile, or a tile looked up ahead, did not change that. 512 experts,
// 1000003 rows, 64 -> 64 half: 24 and 32 us. Quantising the rows in the product's kernel by eight more warps (no second pass over them) took 109 us for that and 258 us for
// the experts before: conversions want the warps of a whole SM.
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

constexpr int PAIR_EXPERTS = 1024;   // whose lists leave shared memory for five stages
constexpr int MX_THREADS = (2 + EPILOGUE_WARPS) * 32, OUT_BYTES = 32 * 128;   // OUT_BYTES: 32 rows x 64 columns of D, per warp of the epilogue

// BN: columns of D; CTAS: blocks that share a tile, each with BM rows of D and BN / CTAS of the columns of B. WHOLE: the kernel quantises its rows itself.
// KB: bytes of a row's codes in a step, 128 (256 channels) or, for matrices of up to 64 channels, 32: stages of a quarter, and more of them.
template <int BN, int CTAS, bool WHOLE, int KB>
struct MxLayout {
    static constexpr int BCOLS = BN / CTAS, ABYTES = BM * KB, BBYTES = BCOLS * KB, BOXBYTES = 64 * KB;
    static constexpr int BTILES = (BN + MX_TILE - 1) / MX_TILE;       // tiles of scales of the columns (each block has all of them)
    static constexpr int SCALES = ABYTES + BBYTES, STAGE = SCALES + SCALE_BYTES * (1 + BTILES);
    // Two blocks per SM for narrow layers: a tile of 128 x 64 and a step or two costs the warp that issues its products more time (1250 clocks to walk on, wait
    // four times and issue) than anything else.
    static constexpr int BLOCKS = BN == 64 && !WHOLE ? 2 : 1, STAGES = KB == 32 ? (BN == 64 ? 7 : 8) : BN == 64 ? (WHOLE ? 6 : 2) : BN == 128 ? 4 : 5, EXPERTS = CTAS == 2 ? PAIR_EXPERTS : EXPERTS_MAX;
    // tensor memory: accumulators, then two sets of scales, used in turn: of 128 rows (4 columns) for two times 128 channels, of the columns likewise
    static constexpr bool OVERLAP = BN == 256;
    static constexpr int SECOND = OVERLAP ? BN - 64 : BN;             // column of the second accumulator
    static constexpr int SCALE_AT = SECOND + BN, SCALE_SET = 32, SCALE_B = 8, SCALE_B_STEP = 4 * BTILES;
    static constexpr int TMEM = SCALE_AT + 2 * SCALE_SET <= 256 ? 256 : 512;
    static constexpr int OUT = STAGES * STAGE, BIAS = OUT + EPILOGUE_WARPS * OUT_BYTES, CONTROL = BIAS + EPILOGUE_WARPS * BN * 4;
    // barriers: full, empty (STAGES each), accumulator full, empty, overlap free (2 each), drain; then flag and tensor memory
    static constexpr int FULL = 0, EMPTY = 64, ACC_FULL = 128, ACC_EMPTY = 144, SHARED_FREE = 160, DRAIN = 176, FAILED = 184, BASE = 188, BARS = 192;
    // 1 KB for the alignment of the ring
    static constexpr int bytes(int experts) { return 1024 + CONTROL + BARS + listInts(experts) * 4; }
    static_assert(SCALE_AT + 2 * SCALE_SET <= TMEM && SCALE_B + 2 * SCALE_B_STEP <= SCALE_SET, "tensor memory");
    static_assert(STAGE % 1024 == 0 && STAGES <= 8, "ring");
    static_assert(BLOCKS * (bytes(EXPERTS) + 1536) <= 228 * 1024, "shared memory");
};

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
// Tells the leader that tensor memory was read. Relaxed: what was read is in registers (tcgen05.wait::ld), and a release would wait for the warp's stores of
// D as well, which took a microsecond per tile (16 experts, 131072 rows, 1024 -> 1024 bfloat16: 111 us for the product, 90 us without).
__device__ __forceinline__ void clusterArriveRelaxed(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// descriptor of a 32-byte swizzled K-major operand: groups of 8 rows of 32 bytes
__device__ __forceinline__ uint64_t narrowDescriptor(uint32_t address)
{
    return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (1ull << 16) | (16ull << 32) | (1ull << 46) | (6ull << 61);
}
// descriptor of a tile of scales: no swizzle, groups of 8 rows of 16 bytes lie 128 bytes apart
__device__ __forceinline__ uint64_t scaleDescriptor(uint32_t address) { return static_cast<uint64_t>((address >> 4) & 0x3FFFu) | (8ull << 32) | (1ull << 46); }

// ---- the rows in 4 bits ----------------------------------------------------------------------------------------------------
// Tiles of 128 rows of one expert, in the order of the product's units (of tileRows rows): tile t of all is part t % (tileRows / 128) of unit t / (tileRows / 128).
// First row and rows of every tile (`piece` rows, or what is left), a thread each; where the experts' units begin, if `unitsBefore` is given. (A block of the
// quantisation that looks for its tile's expert itself has to add up the offsets first: as persistent blocks, which do it once, that kernel took 103 us for 131072
// rows of 1024 bfloat16, a block per tile with this list 73 us, and 55 us with loads that depend on no condition.)
__global__ void __launch_bounds__(TILE_THREADS) mx_tiles_kernel(const __grid_constant__ ProductArgs p, int2* __restrict__ list, int tiles, int piece,
                                                                int* __restrict__ unitsBefore)
{
    extern __shared__ int lists[];
    chained();
    int *bounds = lists, *before = lists + listStride(p.experts);
    planExperts<FORWARD>(p, bounds, before, nullptr, TILE_THREADS);
    __syncthreads();
    const int tile = blockIdx.x * TILE_THREADS + threadIdx.x, parts = p.tileRows / piece, unit = tile / parts;
    if (unitsBefore != nullptr && blockIdx.x == 0)
        for (int e = threadIdx.x; e <= p.experts; e += TILE_THREADS) unitsBefore[e] = before[e];
    if (tile >= tiles) return;
    int2 found = {0, 0};
    if (unit < before[p.experts]) {
        int low = 0, high = p.experts;   // the last expert whose units begin at or before this one (experts without units end up in front of it)
        while (high - low > 1) {
            const int middle = (low + high) / 2;
            if (before[middle] <= unit) low = middle;
            else high = middle;
        }
        const long long begin = bounds[low] + static_cast<long long>(unit - before[low]) * p.tileRows + (tile - unit * parts) * piece;
        const long long left = bounds[low + 1] - begin;   // (the second part of a unit may be empty)
        if (left > 0) found = make_int2(static_cast<int>(begin), static_cast<int>(min(left, static_cast<long long>(piece))));
    }
    list[tile] = found;
}
// A block per tile of 128 rows x 128 channels. `list`: mx_tiles_kernel's, or null where the rows are one expert's.
template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_rows_kernel(const int2* __restrict__ list, const T* __restrict__ x, long long stride, long long rows, int channels,
                                                               unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, int chunks, int codeBytes)
{
    __shared__ __align__(16) unsigned char tileScales[MX_TILE_BYTES];
    const unsigned tile = blockIdx.x / static_cast<unsigned>(chunks);
    const int chunk = static_cast<int>(blockIdx.x - tile * chunks);
    chained();
    int2 t;
    if (list != nullptr) t = list[tile];
    else {
        const long long begin = static_cast<long long>(tile) * MX_TILE;
        t = make_int2(static_cast<int>(begin), static_cast<int>(max(0ll, min(static_cast<long long>(MX_TILE), rows - begin))));
    }
    if (t.y == 0) return;
    quantizeTile<T, LANES, ALIGNED>(x + t.x * stride, stride, t.y, chunk, channels, codes + static_cast<long long>(t.x) * codeBytes, codeBytes,
                           scales + static_cast<long long>(blockIdx.x) * MX_TILE_BYTES, tileScales);
}

// ---- epilogue ------------------------------------------------------------------------------------------------------------------
// Writes of D go by TMA, 32 rows x 64 columns (128 bytes of a row) at a time, from shared memory: 131072 rows of 1024 columns through the warps, 64 bytes of a
// row at a time, were written at 3.1 TB/s. Runs that end within 32 rows, and rows that the TMA cannot write, take the other way.
__device__ __forceinline__ void tmaStore(const CUtensorMap* map, int x, int y, uint32_t from)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(from) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tmaStoresRead() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tmaStoresDone() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void tmemWait32(float (&v)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(v[i]));
}
struct OutTile {
    int row, rows, column, columns;   // first row of the warp's 32, how many are to be written; first column, how many are left
    long long stride;
    bool wide;
};
// 64 columns of `rows` rows from a warp's memory (rows of 128 bytes, their 16-byte chunks swizzled as the TMA's) to D where the TMA cannot write: 16 bytes at a time, or
// pairs of elements that begin on 4 bytes, which in rows of an odd address are the second and third, fourth and fifth, ... (20000 rows of 64 experts of 300 -> 777:
// element by element 58 us for the call, so 48 us; 23 us for 776 columns, by TMA.)
template <class T>
__device__ __forceinline__ void storeChunk(const unsigned char* mine, T* out, long long stride, int rows, int columns, bool wide)
{
    const int lane = threadIdx.x & 31;
    auto at = [&](int r, int c) { return mine + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2; };
    if (wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + lane / 8, c = lane % 8 * 8;
            if (r < rows && c < columns) store<T, 8>(out + r * stride + c, load<T, 8>(reinterpret_cast<const T*>(at(r, c))));
        }
        return;
    }
    constexpr int AT_ONCE = 8;   // (all read before the first is written: the compiler has to take either memory for the other)
    for (int first = 0; first < rows; first += AT_ONCE) {
        uint32_t pair[AT_ONCE], before[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int r = first + i, odd = static_cast<int>((reinterpret_cast<uintptr_t>(out + r * stride) >> 1) & 1), c = 2 * lane + odd;
            const uint32_t low = *reinterpret_cast<const unsigned short*>(at(r, c)), high = *reinterpret_cast<const unsigned short*>(at(r, (c + 1) & 63));
            pair[i] = low | high << 16;
            before[i] = *reinterpret_cast<const unsigned short*>(at(r, 0));
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int r = first + i;
            if (r >= rows) break;
            T* row = out + r * stride;
            const int odd = static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 1) & 1), c = 2 * lane + odd;
            // (predicates: the branches that a condition becomes took 150 clocks a row)
            const bool both = c + 1 < min(columns, 64);
            asm volatile("{\n\t.reg .pred p, q, s;\n\t.reg .b16 u, v;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 s, %6, 0;\n\t"
                         "cvt.u16.u32 u, %2;\n\tcvt.u16.u32 v, %3;\n\t@p st.global.b32 [%0], %2;\n\t@q st.global.b16 [%0], u;\n\t@s st.global.b16 [%1], v;\n\t}"
                         ::"l"(row + c), "l"(row), "r"(pair[i]), "r"(before[i]), "r"(static_cast<int>(both)), "r"(static_cast<int>(!both && c < columns)),
                         "r"(static_cast<int>(odd != 0 && lane == 0)) : "memory");
        }
    }
}

// A warp's 32 lanes of an accumulator of BN columns from `from` on, plus a bias. `sharedLast`: the last 64 columns first (those that the other accumulator begins
// with); `read` is called when the first 64 are.
template <class T, int BN, class F>
__device__ __forceinline__ void storeAccumulator(uint32_t from, bool sharedLast, const CUtensorMap* map, T* out, const OutTile& o, unsigned char* mine, const float* bias, F&& read)
{
    const int lane = threadIdx.x & 31;
    const bool whole = o.wide && o.rows >= 32;
    constexpr bool EARLY = BN == 256;   // all 64 columns at once, so that `read` comes early (of 64 columns in all, nothing waits for it, and registers are short)
#pragma unroll 1
    for (int i = 0; i < BN / 64; ++i) {
        const int c = (sharedLast ? (i + BN / 64 - 1) % (BN / 64) : i) * 64;
        const bool used = c < o.columns && o.rows > 0;
        if (used) {
            if (lane == 0) tmaStoresRead();   // what was written from this memory last
            __syncwarp();
            float both64[2][32];
            if constexpr (EARLY) {
                tmemLoad32(from + c, both64[0]);
                tmemLoad32(from + c + 32, both64[1]);
                tmemWait(both64[0], both64[1]);
                if (i == 0) read();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[32];
                if constexpr (EARLY) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = both64[h][j];
                } else {
                    tmemLoad32(from + c + h * 32, v);
                    tmemWait32(v);
                    if (h == 1 && i == 0) read();
                }
                const int c0 = c + h * 32;
                if (bias != nullptr) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(bias + c0 + j);
                        v[j] += f.x;
                        v[j + 1] += f.y;
                        v[j + 2] += f.z;
                        v[j + 3] += f.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    store<T, 8>(reinterpret_cast<T*>(mine + lane * 128 + (((h * 4 + j) ^ (lane & 7)) << 4)), pack<T, 8>(*reinterpret_cast<const float (*)[8]>(&v[j * 8])));
            }
            if (whole) {
                fenceProxyAsync();
                __syncwarp();
                if (lane == 0) tmaStore(map, o.column + c, o.row, smemAddress(mine));
            } else {
                __syncwarp();
                storeChunk<T>(mine, out + static_cast<long long>(o.row) * o.stride + o.column + c, o.stride, min(o.rows, 32), o.columns - c, o.wide);
                __syncwarp();
            }
        } else if (i == 0) {
            read();
        }
    }
}

// ---- the product -------------------------------------------------------------------------------------------------------------
// Rows that the kernel quantises itself (see forward()): x, its row stride, whether 16-byte accesses read it
template <class T>
struct RawRows {
    const T* x;
    long long stride;
    bool aligned;
};
// 128 rows x 256 channels of a step by the epilogue's warps, to a stage's codes (128-byte swizzled) and scales
// (LANES threads to a row: 16, fewer where a row has no more than 128 or 64 channels)
template <class T, bool ALIGNED, int LANES>
__device__ __forceinline__ void quantizeStep(const T* x, long long stride, int rows, int channels, int step, unsigned char* codes, unsigned char* scales)
{
    constexpr int THREADS = EPILOGUE_WARPS * 32, ROWS = THREADS / LANES, AT_ONCE = BM / ROWS < 4 ? BM / ROWS : 4;
    const int thread = threadIdx.x - 64, part = thread % LANES, first = thread / LANES, c = step * STEP_CHANNELS + part * SIXTEEN, left = channels - c;
    for (int begin = 0; begin < rows; begin += ROWS * AT_ONCE) {   // (rows that are not there: whatever, their rows of D are not stored)
        Sixteen<T> v[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) v[i] = loadSixteen<T, ALIGNED>(x + min(begin + i * ROWS + first, rows - 1) * stride + (left > 0 ? c : 0), left);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int r = begin + i * ROWS + first;
            if (begin + i * ROWS >= rows) break;
            trim<T, ALIGNED>(v[i], left);
            uint32_t largest = largestOf<T>(v[i]);
            largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            const uint32_t scale = scaleOf(largest);
            *reinterpret_cast<uint2*>(codes + r * 128 + ((part / 2 ^ (r & 7)) << 4) + (part & 1) * 8) = encodeSixteen<T>(v[i], scale);
            if ((part & 1) == 0) scales[part / 8 * MX_TILE_BYTES + (r & 31) * 16 + (r >> 5) * 4 + part / 2 % 4] = static_cast<unsigned char>(scale);
        }
    }
}

template <class T, int BN, int CTAS, bool WHOLE, int KB>
__global__ void __launch_bounds__(MX_THREADS, MxLayout<BN, CTAS, WHOLE, KB>::BLOCKS)
    mx_product_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const __grid_constant__ CUtensorMap mapScaleA,
                      const __grid_constant__ CUtensorMap mapScaleB, const __grid_constant__ CUtensorMap mapOut, const __grid_constant__ ProductArgs p, int chunks, const __grid_constant__ RawRows<T> raws)
{
    static_assert(!WHOLE || (CTAS == 1 && KB == 128), "");
    using L = MxLayout<BN, CTAS, WHOLE, KB>;
    extern __shared__ unsigned char dynamic[];
    const uint32_t raw = smemAddress(dynamic), ring = (raw + 1023u) & ~1023u;
    unsigned char* base = dynamic + (ring - raw);
    unsigned char* control = base + L::CONTROL;
    const uint32_t bars = ring + L::CONTROL;
    const uint32_t full = bars + L::FULL, empty = bars + L::EMPTY, accFull = bars + L::ACC_FULL, accEmpty = bars + L::ACC_EMPTY, sharedFree = bars + L::SHARED_FREE;
    volatile int* failed = reinterpret_cast<volatile int*>(control + L::FAILED);
    uint32_t* tmemBase = reinterpret_cast<uint32_t*>(control + L::BASE);
    int *bounds = reinterpret_cast<int*>(control + L::BARS), *before = bounds + listStride(p.experts);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 1 ? 0u : clusterRank();

    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            barrierInit(full + s * 8, WHOLE ? 1 + EPILOGUE_WARPS : CTAS);
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
    const int steps = KB == 32 ? 1 : (p.sum + STEP_CHANNELS - 1) / STEP_CHANNELS;
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
            const int boxesA = WHOLE ? 0 : boxes(t.end - row, BM / 64), boxesB = boxes(p.columns - column, L::BCOLS / 64);
            const uint32_t bytes = (boxesA + boxesB) * L::BOXBYTES + SCALE_BYTES * ((WHOLE ? 0 : 1) + L::BTILES);   // of this block; of both blocks:
            const uint32_t allBytes = CTAS == 1 ? bytes : bytes + (boxes(t.end - row - BM, BM / 64) + boxes(p.columns - column - L::BCOLS, L::BCOLS / 64)) * L::BOXBYTES + SCALE_BYTES * (1 + L::BTILES);
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
                if constexpr (!WHOLE) {
#pragma unroll
                    for (int i = 0; i < BM / 64; ++i) tmaLoad2<CTAS>(lead && i < boxesA, a + i * L::BOXBYTES, &mapA, k * 32, row + i * 64, ready);
                    tmaLoad2<CTAS>(lead, s, &mapScaleA, 0, scaleA + k * 2, ready);
                }
#pragma unroll
                for (int i = 0; i < L::BCOLS / 64; ++i) tmaLoad3<CTAS>(lead && i < boxesB, b + i * L::BOXBYTES, &mapB, k * 32, column + i * 64, t.expert, ready);
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
            const uint32_t columnsAt = BN < MX_TILE ? t.column % MX_TILE / 32 : 0;   // (a tile of 64 columns has half a tile of scales)
            for (int k = 0; __all_sync(0xffffffffu, k < steps); ++k) {
                if (!await(full + stage * 8, phase, failed)) { ok = false; break; }
                // the products that read this set of scales are done (those of the step before keep the tensor core busy meanwhile)
                if (before2 != 0 && !await(before2 & 0x7fffffffu, before2 >> 31, failed)) { ok = false; break; }
                fenceAfter();
                const uint32_t a = ring + stage * L::STAGE, b = a + L::ABYTES, s = a + L::SCALES, scales = tmem + L::SCALE_AT + set * L::SCALE_SET;
                const int parts = min(STEP_CHANNELS, p.sum - k * STEP_CHANNELS + 63) / 64;
                const uint64_t descA = KB == 32 ? narrowDescriptor(a) : operandDescriptor(a, 16), descB = KB == 32 ? narrowDescriptor(b) : operandDescriptor(b, 16), descS = scaleDescriptor(s);
#pragma unroll
                for (int c = 0; c < (KB == 32 ? 1 : 2); ++c) {
                    copyScales<CTAS>(lead && parts > 2 * c, scales + c * 4, descS + c * (MX_TILE_BYTES >> 4));
#pragma unroll
                    for (int i = 0; i < L::BTILES; ++i)
                        copyScales<CTAS>(lead && parts > 2 * c, scales + L::SCALE_B + c * L::SCALE_B_STEP + i * 4, descS + ((SCALE_BYTES * (1 + i) + c * MX_TILE_BYTES) >> 4));
                }
                // 64 channels: 32 bytes of a row, two scales of a word of four
#pragma unroll
                for (int i = 0; i < (KB == 32 ? 1 : 4); ++i)
                    mmaMx<CTAS>(lead && i < parts, d, descA + i * (32 >> 4), descB + i * (32 >> 4), instruction | (i & 1 ? (2u << 29) | (2u << 4) : 0u), scales + i / 2 * 4,
                                scales + L::SCALE_B + i / 2 * L::SCALE_B_STEP + columnsAt, i > 0 ? 1u : k > 0 ? 1u : 0u);
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
        unsigned char* mine = base + L::OUT + (warp - 2) * OUT_BYTES;
        float* mineBias = reinterpret_cast<float*>(base + L::BIAS) + (warp - 2) * BN;
        const uint32_t released = CTAS == 1 ? accEmpty + group * 8 : inBlock(accEmpty + group * 8, 0);
        const uint32_t sharedReleased = CTAS == 1 ? sharedFree + group * 8 : inBlock(sharedFree + group * 8, 0);
        auto release = [&](uint32_t bar) {
            fenceBefore();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CTAS == 1) barrierArrive(bar);
                else clusterArriveRelaxed(bar);
            }
        };
        T* out = static_cast<T*>(p.out);
        uint32_t accPhase = 0, stage = 0, phase = 0, turn = 0;
        if constexpr (!WHOLE) walk = Walk<FORWARD, BN, CTAS>(p, bounds, before, nullptr, group, EPILOGUE_GROUPS);
        bool ok = true;
        while (ok && walk.next(t)) {
            if (t.expert < 0) break;
            if constexpr (WHOLE) {   // the tile's rows, by both groups; then its epilogue, by one
                for (int k = 0; k < steps; ++k) {
                    if (!await(empty + stage * 8, phase ^ 1, failed)) { ok = false; break; }
                    unsigned char* codes = base + stage * L::STAGE;
                    const T* x = raws.x + static_cast<long long>(t.begin) * raws.stride;
                    auto quantize = [&](auto aligned) {
                        constexpr bool A = decltype(aligned)::value;
                        if (p.sum <= 64) quantizeStep<T, A, 4>(x, raws.stride, t.end - t.begin, p.sum, k, codes, codes + L::SCALES);
                        else if (p.sum <= 128) quantizeStep<T, A, 8>(x, raws.stride, t.end - t.begin, p.sum, k, codes, codes + L::SCALES);
                        else quantizeStep<T, A, 16>(x, raws.stride, t.end - t.begin, p.sum, k, codes, codes + L::SCALES);
                    };
                    if (raws.aligned) quantize(std::true_type());
                    else quantize(std::false_type());
                    fenceProxyAsync();
                    __syncwarp();
                    if (lane == 0) barrierArrive(full + stage * 8);
                    if (++stage == L::STAGES) { stage = 0; phase ^= 1; }
                }
                if (!ok || (turn++ & 1) != static_cast<uint32_t>(group)) continue;
            }
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
            storeAccumulator<T, BN>(tmem + group * L::SECOND + (static_cast<uint32_t>(quarter * 32) << 16), L::OVERLAP && group == 0, &mapOut, out,
                                    {tileRow + quarter * 32, t.end - tileRow - quarter * 32, t.column, p.columns - t.column, p.outStride, p.wideStore}, mine,
                                    p.bias != nullptr ? mineBias : nullptr, [&] { if (L::OVERLAP) release(sharedReleased); });
            release(released);
        }
        // rows before the first and behind the last expert belong to nobody
        const int first = bounds[0], last = bounds[p.experts];
        const long long warps = static_cast<long long>(gridDim.x) * EPILOGUE_WARPS, me = static_cast<long long>(blockIdx.x) * EPILOGUE_WARPS + (warp - 2);
        for (long long r = me; r < first + (p.rows - last); r += warps) {
            T* row = out + (r < first ? r : last + (r - first)) * p.outStride;
            for (int c = lane; c < p.columns; c += 32) row[c] = Element<T>::from(0.f);
        }
        if (lane == 0) tmaStoresDone();
        __syncwarp();
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

// ---- few rows: matrix-vector products -----------------------------------------------------------------------------------------
// The product of a handful of rows is bound by reading their experts' matrices. blockIdx.y is a row; its warps take 4 channels out each, those whose scales share 16
// bytes of a tile: n, n + 32, n + 64, n + 96; `split` of them share these where the matrix' rows are long. A lane takes blocks of 32 channels: 16 bytes of codes.
// Codes become pairs of halves, one instruction a pair, and so did the row's: products of e2m1 numbers are multiples of 1/4 up to 36, so that 8 of them are added up in
// half without a rounding; from there on in fp32, times two powers of two. The first codes are asked for before the row is quantised. Rows of one expert read its matrix
// each for itself (from L2, but for the first): blocks of up to 4 rows that share their reads took longer, 16 rows of 1024 -> 1024 9.5 us, now 6.9, 4 of 4096 -> 4096 14.6 us,
// now 13.1. One row of 4096 -> 4096, 9 MB from memory: 6.6 us, 4 of them before the first byte comes; a way over bytes, twice a code's value looked up in registers, and
// dp4a 8.3 us.
constexpr int FEW_WARPS = 8, FEW_OUT = 4, PLANES = MX_BLOCK / 8;   // PLANES: of 8 channels, 16 bytes as halves
// eight codes to four pairs of halves
__device__ __forceinline__ void decodePairs(uint32_t codes, __half2* h)
{
    uint32_t u[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(codes));
    memcpy(h, u, sizeof(u));
}
constexpr int NO_SCALE = 1 << 12;   // in the place of a row's scale 255
// sum * 2^(a + b - 254) for a row's scale a and a matrix' b, NaN if one of them is
__device__ __forceinline__ float scaled(float sum, int a, uint32_t b)
{
    const int e = a + static_cast<int>(b) - 127;
    if (static_cast<unsigned>(e - 1) < 254u && b != 255) return sum * __uint_as_float(static_cast<uint32_t>(e) << 23);
    if (a == NO_SCALE || b == 255) return __uint_as_float(0x7fffffffu);
    // in two steps: a power alone is out of range where the product need not be (below 4, nothing is left of any sum)
    const int two = max(e + 127, 4);
    return sum * __uint_as_float(static_cast<uint32_t>(two / 2) << 23) * __uint_as_float(static_cast<uint32_t>(two - two / 2) << 23);
}

template <class T, bool ALIGNED>
__global__ void __launch_bounds__(FEW_WARPS * 32, 2) mx_few_rows_kernel(const __grid_constant__ MxLinearArgs a, int codeBytes, int chunks, int split)
{
    extern __shared__ uint4 quantized[];   // planes x blocks, 8 halves each; then the blocks' scales
    __shared__ int found;
    __shared__ float sums[FEW_WARPS][FEW_OUT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y, experts = static_cast<int>(a.weight.matrices), columns = static_cast<int>(a.weight.rows);
    const int channels = a.weight.channels, blocks = codeBytes / 16;
    const int group = blockIdx.x * (FEW_WARPS / split) + warp / split, within = group % 32, tile = group / 32, first = tile * MX_TILE + within;   // channels out: first + 32 q
    T* y = static_cast<T*>(a.y.data);
    chained();
    int expert = 0;
    if (a.offsets != nullptr) {
        if (threadIdx.x == 0) found = experts + 1;
        __syncthreads();
        // the first offset behind the row ends its expert's run (offsets are their running maximum): that expert is the one before it
        int behind = experts + 1;
        for (int e = threadIdx.x; e <= experts; e += FEW_WARPS * 32)
            if (a.offsets[e] > row) { behind = e; break; }
        if (behind <= experts) atomicMin(&found, behind);
        __syncthreads();
        behind = found;
        if (behind == 0 || behind > experts) {   // nobody's row
            if (warp % split == 0 && lane < FEW_OUT && first + lane * 32 < columns) y[row * a.y.stride + first + lane * 32] = Element<T>::from(0.f);
            return;
        }
        expert = behind - 1;
    }
    // codes and scales of a block of the warp's channels out (channels and blocks that are not there: the last ones again, and not used)
    const unsigned char* codes[FEW_OUT];
#pragma unroll
    for (int q = 0; q < FEW_OUT; ++q) codes[q] = a.weight.codes + (static_cast<long long>(expert) * columns + min(first + q * 32, columns - 1)) * codeBytes;
    const unsigned char* scales = a.weight.scales + (static_cast<long long>(expert) * ((columns + MX_TILE - 1) / MX_TILE) + tile) * chunks * MX_TILE_BYTES + within * 16;
    auto fetch = [&](int block, uint4 (&code)[FEW_OUT], uint4& scale) {
        const int b = min(block, blocks - 1);
        scale = *reinterpret_cast<const uint4*>(scales + static_cast<long long>(b / 4) * MX_TILE_BYTES);
#pragma unroll
        for (int q = 0; q < FEW_OUT; ++q) code[q] = *reinterpret_cast<const uint4*>(codes[q] + b * 16);
    };
    const int begin = warp % split * 32 + lane, step = split * 32;
    uint4 code[2][FEW_OUT], scale[2];   // of this turn and the next
    fetch(begin, code[0], scale[0]);
    fetch(begin + step, code[1], scale[1]);
    // the row: half a block a thread
    int16_t* rowScales = reinterpret_cast<int16_t*>(quantized + PLANES * blocks);
    const T* x = static_cast<const T*>(a.x.data) + row * a.x.stride;
    for (int h = threadIdx.x; h - lane < blocks * 2; h += FEW_WARPS * 32) {
        const int left = channels - h * SIXTEEN;
        Sixteen<T> v = loadSixteen<T, ALIGNED>(x + (left > 0 ? h * SIXTEEN : 0), left);
        trim<T, ALIGNED>(v, left);
        uint32_t largest = largestOf<T>(v);
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        const uint32_t s = scaleOf(largest);
        const uint2 c = encodeSixteen<T>(v, s);
        if (h >= blocks * 2) continue;
        __half2 pairs[8];
        decodePairs(c.x, pairs);
        decodePairs(c.y, pairs + 4);
        uint4 u[2];
        memcpy(u, pairs, sizeof(u));
        quantized[(h & 1) * 2 * blocks + h / 2] = u[0];
        quantized[((h & 1) * 2 + 1) * blocks + h / 2] = u[1];
        if ((h & 1) == 0) rowScales[h / 2] = static_cast<int16_t>(s == 255 ? NO_SCALE : static_cast<int>(s));
    }
    __syncthreads();
    float sum[FEW_OUT] = {};
    auto add = [&](int block, const uint4 (&code)[FEW_OUT], const uint4& scale) {
        const int at = (block & 3) * 8, rowScale = rowScales[block];
        const uint32_t s[FEW_OUT] = {scale.x >> at & 255u, scale.y >> at & 255u, scale.z >> at & 255u, scale.w >> at & 255u};
        float all[FEW_OUT] = {};
#pragma unroll
        for (int p = 0; p < PLANES; p += 2) {   // 16 channels
            const uint4 u[2] = {quantized[p * blocks + block], quantized[(p + 1) * blocks + block]};
            __half2 xs[8];
            memcpy(xs, u, sizeof(u));
#pragma unroll
            for (int q = 0; q < FEW_OUT; ++q) {
                const uint32_t words[PLANES] = {code[q].x, code[q].y, code[q].z, code[q].w};
                __half2 w[8];
                decodePairs(words[p], w);
                decodePairs(words[p + 1], w + 4);
                __half2 h = __hmul2(w[0], xs[0]);
#pragma unroll
                for (int i = 1; i < 8; ++i) h = __hfma2(w[i], xs[i], h);
                const float2 f = __half22float2(h);
                all[q] += f.x + f.y;
            }
        }
#pragma unroll
        for (int q = 0; q < FEW_OUT; ++q) sum[q] += scaled(all[q], rowScale, s[q]);
    };
    for (int block = begin; block - lane < blocks; block += 2 * step) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = block + i * step;
            if (b < blocks) add(b, code[i], scale[i]);
            if (b - lane + 2 * step < blocks) fetch(b + 2 * step, code[i], scale[i]);
        }
    }
    // lane q keeps that sum; then the warps that share channels out join theirs
    float mine = 0.f;
#pragma unroll
    for (int q = 0; q < FEW_OUT; ++q) {
        const float all = groupSum<32>(sum[q]);
        mine = lane == q ? all : mine;
    }
    if (split > 1) {
        if (lane < FEW_OUT) sums[warp][lane] = mine;
        __syncthreads();
        if (warp % split != 0) return;
        mine = 0.f;
        if (lane < FEW_OUT)
            for (int w = 0; w < split; ++w) mine += sums[warp + w][lane];
    }
    const int n = first + lane * 32;
    if (lane < FEW_OUT && n < columns) {
        const float b = a.bias != nullptr ? Element<T>::to(static_cast<const T*>(a.bias)[static_cast<long long>(expert) * columns + n]) : 0.f;
        y[row * a.y.stride + n] = Element<T>::from(mine + b);
    }
}

// ---- bias gradient without an input gradient: column sums of an expert's rows --------------------------------------------------------------------------------
// Pieces of BIAS_ROWS rows of one expert and 64 columns (32 element by element) a block, joined in order. 131072 rows of 1024 bfloat16, 16 experts: 57 us (a block
// per expert and 32 columns 199 us).
constexpr int BIAS_ROWS = 1024, BIAS_THREADS = 256;
template <int VEC> constexpr int BIAS_LANES = VEC == 8 ? 8 : 32;
template <class T, int VEC>
__global__ void __launch_bounds__(BIAS_THREADS) mx_bias_kernel(const int2* __restrict__ list, const T* __restrict__ dy, long long stride, int columns, float* __restrict__ partial)
{
    constexpr int LANES = BIAS_LANES<VEC>, STEP = BIAS_THREADS / LANES, COLUMNS = LANES * VEC, AT_ONCE = 8;
    __shared__ float sums[BIAS_THREADS / 32][COLUMNS];
    chained();
    const unsigned groups = (columns + COLUMNS - 1) / COLUMNS, piece = blockIdx.x / groups;   // (blocks side by side read the rows' neighbouring columns)
    const int firstColumn = static_cast<int>(blockIdx.x - piece * groups) * COLUMNS;
    const int2 t = list[piece];
    if (t.y == 0) return;
    const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES, c = firstColumn + lane * VEC;
    float sum[VEC] = {};
    if (c < columns) {
        const T* at = dy + (static_cast<long long>(t.x) + first) * stride + c;
        auto add = [&](const Pack<T, VEC>& v) {
            float f[VEC];
            unpack<T, VEC>(v, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[j] += f[j];
        };
        int r = first;
        for (; r + (AT_ONCE - 1) * STEP < t.y; r += STEP * AT_ONCE) {
            Pack<T, VEC> v[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) v[i] = load<T, VEC>(at + i * STEP * stride);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) add(v[i]);
            at += STEP * AT_ONCE * stride;
        }
        for (; r < t.y; r += STEP) {
            add(load<T, VEC>(at));
            at += STEP * stride;
        }
    }
    // the rows of a warp, then the warps
#pragma unroll
    for (int o = LANES; o < 32; o *= 2)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], o);
    if ((threadIdx.x & 31) < LANES) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[threadIdx.x / 32][lane * VEC + j] = sum[j];
    }
    __syncthreads();
    const int column = firstColumn + threadIdx.x;
    if (threadIdx.x < COLUMNS && column < columns) {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < BIAS_THREADS / 32; ++i) all += sums[i][threadIdx.x];
        partial[static_cast<long long>(piece) * columns + column] = all;
    }
}
// the sums of an expert's pieces, perUnit of them for each of its units, of 32 columns: JOIN_ROWS threads to a column
constexpr int JOIN_ROWS = 16;
template <class T>
__global__ void __launch_bounds__(32 * JOIN_ROWS) mx_bias_join_kernel(const int* __restrict__ unitsBefore, int perUnit, const float* __restrict__ partial, int columns, T* __restrict__ out)
{
    __shared__ float sums[JOIN_ROWS][32];
    chained();
    const int expert = blockIdx.x, lane = threadIdx.x & 31, part = threadIdx.x / 32, c = blockIdx.y * 32 + lane;
    const long long end = static_cast<long long>(unitsBefore[expert + 1]) * perUnit;
    float sum = 0.f;
    if (c < columns) {
#pragma unroll 8
        for (long long u = static_cast<long long>(unitsBefore[expert]) * perUnit + part; u < end; u += JOIN_ROWS) sum += partial[u * columns + c];
    }
    sums[part][lane] = sum;
    __syncthreads();
    if (part == 0 && c < columns) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < JOIN_ROWS; ++i) sum += sums[i][lane];
        out[static_cast<long long>(expert) * columns + c] = Element<T>::from(sum);
    }
}

// ---- input gradient of half rows where half does not hold a matrix -------------------------------------------------------------
// Matrices whose powers of two lie between -13 and 13 are decoded to half as they are; others are divided by a power of two, which the product's sums are multiplied
// with in fp32 (mx_ranges_kernel, dividedBy). What remains are matrices whose blocks lie more than 2^26 apart: their rows of dx are computed once more here,
// dx_rc = sum over n of dy_rn (W_nc 2^E), codes decoded to fp32, sums in fp32. Few weights look like that, so this kernel is plain: a tile of 128 rows x 64 channels in
// a block, 32 channels out at a time through shared memory. 131072 rows of half, 16 experts of 1024 -> 1024: 182 us where no matrix is apart, 815 with one of the 16, 8.6 ms with all;
// finding it out costs every call of half rows 3 to 6 us (2.5 to 5 in front, less for small matrices, and 2 for this kernel's launch).
constexpr int APART_COLUMNS = 64, APART_STEP = 32, APART_THREADS = 256;
__global__ void __launch_bounds__(APART_THREADS) mx_apart_kernel(const __grid_constant__ ProductArgs p, const __grid_constant__ MxMatrix w, const int* __restrict__ apart,
                                                                 const __half* __restrict__ dy, long long stride, int codeBytes, int chunks)
{
    extern __shared__ int lists[];
    __shared__ float rows[APART_STEP][BM + 1];
    __shared__ __align__(16) float columns[APART_STEP][APART_COLUMNS];
    chained();
    int any = 0;
    for (int e = threadIdx.x; e < p.experts; e += APART_THREADS) any |= apart[e];
    if (!__syncthreads_or(any)) return;
    int *bounds = lists, *before = lists + listStride(p.experts);
    planExperts<FORWARD>(p, bounds, before, nullptr, APART_THREADS);
    __syncthreads();
    Walk<FORWARD, APART_COLUMNS, 1> walk(p, bounds, before, nullptr, 0, 1);
    Tile t;
    const int line = threadIdx.x / 32, lane = threadIdx.x & 31, mine = threadIdx.x / 16 * 8, column = threadIdx.x % 16 * 4;   // 8 rows x 4 channels of a thread
    const int channelsOut = static_cast<int>(w.rows), tilesOut = (channelsOut + MX_TILE - 1) / MX_TILE;
    while (walk.next(t)) {
        if (t.expert < 0) break;
        if (apart[t.expert] == 0) continue;
        float sum[8][4] = {};
        for (int begin = 0; begin < channelsOut; begin += APART_STEP) {
#pragma unroll 4
            for (int r = line; r < BM; r += APART_THREADS / 32) {
                const bool there = r < t.end - t.begin && begin + lane < channelsOut;
                rows[lane][r] = there ? __half2float(dy[(static_cast<long long>(t.begin) + r) * stride + begin + lane]) : 0.f;
            }
            {   // 8 channels of a channel out
                const int k = threadIdx.x / 8, n = begin + k, c = t.column + threadIdx.x % 8 * 8;
                float f[8] = {};
                if (n < channelsOut && c / 2 < codeBytes) {
                    const long long matrix = t.expert;
                    const unsigned char scale = w.scales[((matrix * tilesOut + n / MX_TILE) * chunks + c / MX_TILE) * MX_TILE_BYTES + n % 32 * 16 + n % MX_TILE / 32 * 4 + c % MX_TILE / MX_BLOCK];
                    decodeEight(*reinterpret_cast<const uint32_t*>(w.codes + (matrix * channelsOut + n) * codeBytes + c / 2), f);
                    const float power = powerOf(scale);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] *= power;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) columns[k][threadIdx.x % 8 * 8 + i] = f[i];
            }
            __syncthreads();
#pragma unroll 4
            for (int k = 0; k < APART_STEP; ++k) {
                const float4 b = *reinterpret_cast<const float4*>(&columns[k][column]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = rows[k][mine + i];
                    sum[i][0] += a * b.x;
                    sum[i][1] += a * b.y;
                    sum[i][2] += a * b.z;
                    sum[i][3] += a * b.w;
                }
            }
            __syncthreads();
        }
        __half* out = static_cast<__half*>(p.out);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (mine + i < t.end - t.begin && t.column + column + j < p.columns)
                    out[(static_cast<long long>(t.begin) + mine + i) * p.outStride + t.column + column + j] = __float2half_rn(sum[i][j]);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// an encoding, once more with a context: in a thread's first call the driver wants one, which the runtime binds
template <class F>
cudaError_t encoded(F&& run)
{
    if (encoder() == nullptr) return cudaErrorNotSupported;
    CUresult r = run();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess) e = cudaSetDevice(device);
        if (e != cudaSuccess) return e;
        r = run();
    }
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
// `matrices` matrices of `rows` rows of `bytes` bytes, one behind the other (0: one, for a 2-D map), boxes of boxRows x boxBytes
cudaError_t encodeBytes(CUtensorMap& map, const void* data, long long matrices, long long rows, int bytes, int boxBytes, int boxRows, CUtensorMapSwizzle swizzle)
{
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(bytes / 4), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(matrices)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(bytes), static_cast<cuuint64_t>(bytes) * rows};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(boxBytes / 4), static_cast<cuuint32_t>(boxRows), 1}, one[3] = {1, 1, 1};
    return encoded([&] {
        return encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, matrices > 0 ? 3 : 2, const_cast<void*>(data), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}
// rows of D, boxes of 32 x 64 elements of 16 bits
cudaError_t encodeOut(CUtensorMap& map, void* data, long long rows, int columns, long long stride)
{
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[2] = {64, 32}, one[2] = {1, 1};
    return encoded([&] {
        return encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    });
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// One kernel, which quantises a tile's rows itself, where there are no more tiles than SMs and a tile's rows are a few batches of what its threads take at once (64
// rows of 256 channels): a batch costs about a microsecond, the kernels that list and quantise the rows first 4 us with offsets and 2 us without. us, so / with
// those kernels: 16 experts of 256 -> 256, 4 to 512 rows 7.2 to 7.7 / 11.1 to 11.7; 16 of 1024 -> 1024, 4 rows 9.7 / 12.2, 512 rows 12.7 / 12.7; 8 of 4096 -> 1024, 4
// rows 19.5 / 16.2; one of 512 -> 2048, 4 rows 7.7 / 8.7, 128 rows 10.8 / 8.7.
bool wholeRows(const MxLinearArgs& a)
{
    const int lanes = a.weight.channels <= 64 ? 4 : a.weight.channels <= 128 ? 8 : 16, batch = 1024 / lanes, steps = (a.weight.channels + STEP_CHANNELS - 1) / STEP_CHANNELS;
    const long long rows = std::min<long long>((a.rows + a.weight.matrices - 1) / a.weight.matrices, MX_TILE);
    return steps * ((rows + batch - 1) / batch) <= (a.weight.matrices > 1 ? 4 : 2);
}
struct Shape {
    int width, ctas;
    bool whole;   // the product's kernel quantises the rows
};
long long rowTiles(const MxLinearArgs& a, int ctas);
// Pairs of blocks from 512 rows an expert on. us for the call, in pairs / single blocks of 128 columns: 16 experts of 1024 -> 1024, 256 rows each 23.6 / 21.5, 512 rows 25.6 / 25.6, 768 rows
// 29.7 / 31.7, 2048 rows 46 / 52; one of 4096 -> 4096, 512 rows 21.5 / 19.5, 768 rows 21.5 / 25.6; 64 of 512 -> 512, 256 rows 25.6 / 23.6, 512 rows 31.7 / 31.7, 2048 rows 71 / 73.
Shape shapeOf(const MxLinearArgs& a)
{
    const int columns = static_cast<int>(a.weight.rows);
    const long long tiles = rowTiles(a, 1);
    if (wholeRows(a)) {
        if (tiles * ((columns + 63) / 64) <= a.numSMs) return {64, 1, true};
        if (tiles * ((columns + 127) / 128) <= a.numSMs) return {128, 1, true};
    }
    if (columns <= 64) return {64, 1, false};
    if (columns <= 128 || a.rows / a.weight.matrices < 512 || a.weight.matrices > PAIR_EXPERTS) return {128, 1, false};
    return {256, 2, false};
}
// tiles of 128 rows, none with rows of two experts, a multiple of ctas per expert: an upper bound
long long rowTiles(const MxLinearArgs& a, int ctas)
{
    return (a.rows / (MX_TILE * ctas) + std::min<long long>(a.rows, a.weight.matrices)) * ctas;
}
struct MxScratch {
    size_t scales, list, bytes;   // codes lie at the start
    MxScratch(const MxLinearArgs& a)
    {
        const size_t tiles = static_cast<size_t>(rowTiles(a, shapeOf(a).ctas));
        scales = align256(static_cast<size_t>(a.rows) * mxCodeBytes(a.weight.channels));
        list = scales + align256(tiles * mxTiles(a.weight.channels) * MX_TILE_BYTES);
        bytes = list + align256(tiles * sizeof(int2));
    }
};

template <class T>
cudaError_t quantizeRows(const MxLinearArgs& a, const ProductArgs& p, unsigned char* codes, unsigned char* scales, int2* list, cudaStream_t stream)
{
    const int tiles = static_cast<int>(rowTiles(a, p.tileRows / MX_TILE)), chunks = mxTiles(p.sum);
    if (p.offsets != nullptr)
        launchChained(mx_tiles_kernel, (tiles + TILE_THREADS - 1) / TILE_THREADS, TILE_THREADS, 2 * listStride(p.experts) * sizeof(int), stream, 1, p, list, tiles, MX_TILE, static_cast<int*>(nullptr));
    else list = nullptr;
    return byLanes(a.x, a.type, p.sum, [&](auto lanes, auto aligned) {
        launchChained(mx_rows_kernel<T, decltype(lanes)::value, decltype(aligned)::value>, static_cast<unsigned>(tiles) * chunks, TILE_THREADS, 0, stream, 1, list, static_cast<const T*>(a.x.data), a.x.stride,
                      a.rows, p.sum, codes, scales, chunks, mxCodeBytes(p.sum));
        return cudaGetLastError();
    });
}

template <class T, int BN, int CTAS, bool WHOLE, int KB>
cudaError_t launchMx(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& sa, const CUtensorMap& sb, const CUtensorMap& out, const ProductArgs& p, const MxLinearArgs& m,
                     cudaStream_t stream)
{
    using L = MxLayout<BN, CTAS, WHOLE, KB>;
    auto* kernel = mx_product_kernel<T, BN, CTAS, WHOLE, KB>;
    const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), L::bytes(L::EXPERTS));
    if (e != cudaSuccess) return e;
    const RawRows<T> rows = {static_cast<const T*>(m.x.data), m.x.stride, wide(m.x, m.type, p.sum)};
    return launchChained(kernel, m.numSMs / CTAS * CTAS * L::BLOCKS, MX_THREADS, L::bytes(p.experts), stream, CTAS, a, b, sa, sb, out, p, mxTiles(p.sum), rows);
}

// Rows that the matrix-vector kernel takes: as long as its blocks (8 warps, 32 channels out) go over the machine about twice. us, so / by the tensor cores: 1024 ->
// 1024, 16 rows 6.9 / 9.1, 32 rows 11.5 / 9.0; 4096 -> 4096, 3 rows 12.0 / 13.1, 6 rows 18.2 / 13.1; 64 experts of 1024 -> 2048, 12 rows 11.5 / 15.2, 24 rows 19.2 / 16.7;
// 16 of 1024 -> 1024, 24 rows 11.0 / 12.0, 32 rows 14.1 / 12.3; 64 of 256 -> 256, 64 rows 8.4 / 9.1.
int fewGroups(const MxLinearArgs& a) { return mxTiles(a.weight.rows) * 32 / FEW_WARPS; }
int fewBytes(int channels) { return mxBlocks(channels) * (PLANES * 16 + 2); }
bool fewRows(const MxLinearArgs& a)
{
    return a.rows <= 64 && (a.rows == 1 || fewGroups(a) * a.rows <= (a.weight.matrices > 1 ? 768 : 512)) && fewBytes(a.weight.channels) <= 200 * 1024;
}
template <class T>
cudaError_t forwardFewRows(const MxLinearArgs& a, cudaStream_t stream)
{
    // warps that share channels out: as many as there is work for, while all blocks are resident
    const int blocks = mxBlocks(a.weight.channels), groups = fewGroups(a);
    int split = 1;
    while (split < FEW_WARPS && split * 32 < blocks && groups * split * 2 * a.rows <= a.numSMs * 2) split *= 2;
    auto go = [&](auto* kernel) {
        const int bytes = fewBytes(a.weight.channels);
        if (bytes > 47 * 1024) {   // (48 KB without asking, which the kernel's static shared memory counts towards)
            const cudaError_t e = allowShared(reinterpret_cast<const void*>(kernel), 200 * 1024);
            if (e != cudaSuccess) return e;
        }
        launchChained(kernel, dim3(groups * split, static_cast<unsigned>(a.rows)), FEW_WARPS * 32, bytes, stream, 1, a, mxCodeBytes(a.weight.channels), mxTiles(a.weight.channels), split);
        return cudaGetLastError();
    };
    return wide(a.x, a.type, a.weight.channels) ? go(mx_few_rows_kernel<T, true>) : go(mx_few_rows_kernel<T, false>);
}

ProductArgs productArgs(const MxLinearArgs& a, const Shape& shape)
{
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
    return p;
}
// codes, 128 or 32 bytes of a row per box
cudaError_t encodeCodes(CUtensorMap& map, const void* data, long long matrices, long long rows, int bytes, int boxBytes)
{
    return encodeBytes(map, data, matrices, rows, bytes, boxBytes, 64, boxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_32B);
}
cudaError_t encodeWeight(const MxLinearArgs& a, CUtensorMap& map, CUtensorMap& scales, int boxBytes)
{
    const long long tiles = a.weight.matrices * mxTiles(a.weight.rows) * mxTiles(a.weight.channels);
    const cudaError_t e = encodeCodes(map, a.weight.codes, a.weight.matrices, a.weight.rows, mxCodeBytes(a.weight.channels), boxBytes);
    return e != cudaSuccess ? e : encodeBytes(scales, a.weight.scales, 0, tiles, MX_TILE_BYTES, MX_TILE_BYTES, 2, CU_TENSOR_MAP_SWIZZLE_NONE);
}
template <class T>
cudaError_t forward(const MxLinearArgs& a, cudaStream_t stream)
{
    if (fewRows(a)) return forwardFewRows<T>(a, stream);
    const Shape shape = shapeOf(a);
    const MxScratch s(a);
    unsigned char *codes = static_cast<unsigned char*>(a.scratch), *scales = codes + s.scales;
    const ProductArgs p = productArgs(a, shape);
    const int chunks = mxTiles(p.sum), codeBytes = mxCodeBytes(p.sum);
    CUtensorMap mapA = {}, mapB, mapScaleA = {}, mapScaleB, mapOut = {};
    const int boxBytes = !shape.whole && p.sum <= 64 ? 32 : 128;
    cudaError_t e = encodeWeight(a, mapB, mapScaleB, boxBytes);
    if (e == cudaSuccess && p.wideStore) e = encodeOut(mapOut, p.out, a.rows, p.columns, p.outStride);
    if (e != cudaSuccess) return e;
    if (shape.whole)
        return shape.width == 64 ? launchMx<T, 64, 1, true, 128>(mapA, mapB, mapScaleA, mapScaleB, mapOut, p, a, stream)
                                 : launchMx<T, 128, 1, true, 128>(mapA, mapB, mapScaleA, mapScaleB, mapOut, p, a, stream);
    e = encodeCodes(mapA, codes, 0, a.rows, codeBytes, boxBytes);
    if (e == cudaSuccess) e = encodeBytes(mapScaleA, scales, 0, rowTiles(a, shape.ctas) * chunks, MX_TILE_BYTES, MX_TILE_BYTES, 2, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (e == cudaSuccess) e = quantizeRows<T>(a, p, codes, scales, reinterpret_cast<int2*>(codes + s.list), stream);
    if (e != cudaSuccess) return e;
    auto go = [&](auto bytes) {
        constexpr int KB = decltype(bytes)::value;
        if (shape.width == 64) return launchMx<T, 64, 1, false, KB>(mapA, mapB, mapScaleA, mapScaleB, mapOut, p, a, stream);
        if (shape.width == 128) return launchMx<T, 128, 1, false, KB>(mapA, mapB, mapScaleA, mapScaleB, mapOut, p, a, stream);
        return launchMx<T, 256, 2, false, KB>(mapA, mapB, mapScaleA, mapScaleB, mapOut, p, a, stream);
    };
    return boxBytes == 32 ? go(std::integral_constant<int, 32>()) : go(std::integral_constant<int, 128>());
}

// scratch of the adjoint: [units before the experts | the bias gradient's sums | half: how far the matrices' powers of two reach | the matrices in 16 bits | scratch of
// the input gradient's product], or, where the bias gradient is all that is wanted, [units | sums | list of its pieces]
struct MxAdjointScratch {
    size_t partial, found, power, apart, matrices, product, list, bytes;
    int pieces;
    explicit MxAdjointScratch(const MxLinearArgs& a)
    {
        const ExpertArgs r = inputGradient(a);
        pieces = static_cast<int>(a.rows / BIAS_ROWS + std::min<long long>(a.rows, a.weight.matrices));
        partial = align256((static_cast<size_t>(a.weight.matrices) + 1) * sizeof(int));
        found = list = partial + align256(static_cast<size_t>(a.gradX.data != nullptr ? expertSums(r) : pieces) * static_cast<size_t>(a.weight.rows) * sizeof(float));
        const size_t ranges = a.type == TYPE_HALF ? static_cast<size_t>(a.weight.matrices) : 0;
        power = found + align256(ranges * mxRangeParts(a.weight) * sizeof(int2));
        apart = power + align256(ranges * sizeof(float));
        matrices = apart + align256(ranges * sizeof(int));
        product = matrices + (a.gradX.data == nullptr ? 0 : align256(static_cast<size_t>(a.weight.matrices) * a.weight.rows * r.weightStride * 2));
        bytes = a.gradX.data != nullptr ? product + expertBytes(r, true) : list + align256(static_cast<size_t>(pieces) * sizeof(int2));
    }
    // the product with the matrices in 16 bits
    static ExpertArgs inputGradient(const MxLinearArgs& a)
    {
        ExpertArgs r{};
        r.rows = a.rows;
        r.experts = static_cast<int>(a.weight.matrices);
        r.channelsIn = a.weight.channels;
        r.channelsOut = static_cast<int>(a.weight.rows);
        r.type = a.type;
        r.numSMs = a.numSMs;
        r.offsets = a.offsets;
        r.gradY = a.gradY;
        r.gradX = a.gradX;
        r.status = a.status;
        r.weightStride = (r.channelsIn + 7) / 8 * 8;   // (rows that the product's TMA reads as they are: 32 matrices of 300 x 777 decoded in 7 us, else 14 and 9 more for a copy)
        return r;
    }
};
cudaError_t launchApart(const MxLinearArgs& a, const MxRanges& ranges, cudaStream_t stream)
{
    ProductArgs p{};
    p.rows = a.rows;
    p.experts = static_cast<int>(a.weight.matrices);
    p.columns = a.weight.channels;
    p.columnTiles = (p.columns + APART_COLUMNS - 1) / APART_COLUMNS;
    p.tileRows = BM;
    p.offsets = a.offsets;
    p.out = a.gradX.data;
    p.outStride = a.gradX.stride;
    launchChained(mx_apart_kernel, 2 * a.numSMs, APART_THREADS, 2 * listStride(p.experts) * sizeof(int), stream, 1, p, a.weight, ranges.apart, static_cast<const __half*>(a.gradY.data),
                  a.gradY.stride, mxCodeBytes(p.columns), mxTiles(p.columns));
    return cudaGetLastError();
}
template <class T>
cudaError_t joinBias(const MxLinearArgs& a, const MxAdjointScratch& s, int perUnit, cudaStream_t stream)
{
    const int columns = static_cast<int>(a.weight.rows);
    const unsigned char* base = static_cast<const unsigned char*>(a.scratch);
    launchChained(mx_bias_join_kernel<T>, dim3(static_cast<unsigned>(a.weight.matrices), (columns + 31) / 32), 32 * JOIN_ROWS, 0, stream, 1, reinterpret_cast<const int*>(base), perUnit,
                  reinterpret_cast<const float*>(base + s.partial), columns, static_cast<T*>(a.gradBias));
    return cudaGetLastError();
}
// the bias gradient alone
template <class T>
cudaError_t biasGradient(const MxLinearArgs& a, const MxAdjointScratch& s, cudaStream_t stream)
{
    const int columns = static_cast<int>(a.weight.rows), experts = static_cast<int>(a.weight.matrices);
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    auto *list = reinterpret_cast<int2*>(base + s.list);
    auto *before = reinterpret_cast<int*>(base);
    auto *partial = reinterpret_cast<float*>(base + s.partial);
    ProductArgs p{};
    p.rows = a.rows;
    p.experts = experts;
    p.offsets = a.offsets;
    p.tileRows = BIAS_ROWS;
    launchChained(mx_tiles_kernel, (s.pieces + TILE_THREADS - 1) / TILE_THREADS, TILE_THREADS, 2 * listStride(experts) * sizeof(int), stream, 1, p, list, s.pieces, BIAS_ROWS, before);
    const cudaError_t e = byAccess<T>({&a.gradY}, a.type, columns, [&](auto vec) {
        constexpr int VEC = decltype(vec)::value, COLUMNS = BIAS_LANES<VEC> * VEC;
        launchChained(mx_bias_kernel<T, VEC>, static_cast<unsigned>(s.pieces) * ((columns + COLUMNS - 1) / COLUMNS), BIAS_THREADS, 0, stream, 1, list, static_cast<const T*>(a.gradY.data), a.gradY.stride,
                      columns, partial);
        return cudaGetLastError();
    });
    return e != cudaSuccess ? e : joinBias<T>(a, s, 1, stream);
}

} // namespace

size_t mxLinearBytes(const MxLinearArgs& a) { return a.rows == 0 || fewRows(a) || shapeOf(a).whole ? 0 : MxScratch(a).bytes; }
size_t mxLinearAdjointBytes(const MxLinearArgs& a) { return a.rows == 0 ? 0 : MxAdjointScratch(a).bytes; }

cudaError_t launchMxLinear(const MxLinearArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return cudaSuccess;
    return a.type == TYPE_HALF ? forward<__half>(a, stream) : forward<__nv_bfloat16>(a, stream);
}
cudaError_t launchMxLinearAdjoint(const MxLinearArgs& a, cudaStream_t stream)
{
    if (a.rows == 0) return a.gradBias == nullptr ? cudaSuccess : cudaMemsetAsync(a.gradBias, 0, static_cast<size_t>(a.weight.matrices) * a.weight.rows * 2, stream);
    const MxAdjointScratch s(a);
    if (a.gradX.data == nullptr) {
        if (a.gradBias == nullptr) return cudaSuccess;
        return a.type == TYPE_HALF ? biasGradient<__half>(a, s, stream) : biasGradient<__nv_bfloat16>(a, s, stream);
    }
    unsigned char* base = static_cast<unsigned char*>(a.scratch);
    const bool half = a.type == TYPE_HALF;
    const MxRanges ranges = {mxRangeParts(a.weight), reinterpret_cast<int2*>(base + s.found), reinterpret_cast<float*>(base + s.power), reinterpret_cast<int*>(base + s.apart)};
    ExpertArgs r = MxAdjointScratch::inputGradient(a);
    const MxWanted wanted = {a.offsets, a.rows, true};
    cudaError_t e = half ? launchMxRanges(a.weight, wanted, ranges, stream) : cudaSuccess;
    if (e == cudaSuccess) e = launchMxDequantize(a.weight, a.type, {base + s.matrices, r.weightStride}, stream, wanted, half ? &ranges : nullptr);
    if (e != cudaSuccess) return e;
    // the product's tiles of dy lie in shared memory: their columns are added up there
    r.weight = base + s.matrices;
    r.scratch = base + s.product;
    if (a.gradBias != nullptr) {
        r.columnSums = reinterpret_cast<float*>(base + s.partial);
        r.unitsBefore = reinterpret_cast<int*>(base);
    }
    if (half) r.powers = ranges.power;
    e = launchExpertAdjoint(r, stream);
    if (e == cudaSuccess && half) e = launchApart(a, ranges, stream);
    if (e != cudaSuccess || a.gradBias == nullptr) return e;
    return a.type == TYPE_HALF ? joinBias<__half>(a, s, expertSumsPerUnit(r), stream) : joinBias<__nv_bfloat16>(a, s, expertSumsPerUnit(r), stream);
}

} // namespace kernel
} // namespace qmlp
