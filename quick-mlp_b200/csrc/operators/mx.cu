// Matrices to microscaled 4-bit floating point and back (formats: mx.cuh). A block takes a tile of 128 rows x 128 channels, whose scales are one run of 512
// bytes; both directions are bound by memory.
#include "mx.cuh"

namespace qmlp {
namespace kernel {
namespace {

using namespace mx;

// first row and rows of tile `tile` of all matrices' row tiles
struct RowTile {
    long long row;
    int rows;
};
__device__ __forceinline__ RowTile rowTile(const MxMatrix& q, int tilesPerMatrix, unsigned tile)
{
    const unsigned matrix = static_cast<unsigned>(tile) / static_cast<unsigned>(tilesPerMatrix);
    const long long within = static_cast<long long>(static_cast<unsigned>(tile) - matrix * tilesPerMatrix) * MX_TILE;
    return {matrix * q.rows + within, static_cast<int>(min(static_cast<long long>(MX_TILE), q.rows - within))};
}

template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_quantize_kernel(const __grid_constant__ MxMatrix q, const T* __restrict__ x, long long stride, int tilesPerMatrix, int chunks,
                                                                   int codeBytes)
{
    chained();
    __shared__ __align__(16) unsigned char tileScales[MX_TILE_BYTES];
    const unsigned tile = blockIdx.x / static_cast<unsigned>(chunks);
    const int chunk = static_cast<int>(blockIdx.x - tile * chunks);
    const RowTile t = rowTile(q, tilesPerMatrix, tile);
    quantizeTile<T, LANES, ALIGNED>(x + t.row * stride, stride, t.rows, chunk, q.channels, q.codes + t.row * codeBytes, codeBytes,
                                    q.scales + static_cast<long long>(blockIdx.x) * MX_TILE_BYTES, tileScales);
}

// An expert whose offsets, taken as they are used (within [0, rows], their running maximum), do not rise has no rows. (They rise only where they rise here.)
__device__ __forceinline__ bool hasRows(const MxWanted& w, unsigned matrix)
{
    if (w.offsets == nullptr) return true;
    const long long begin = max(w.offsets[matrix], 0), end = w.offsets[matrix + 1];
    return min(end, w.rows) > min(begin, w.rows);
}

// The lowest and highest power of two (+ 127) of blocks of a matrix, from their scales: those of the tiles first, first + step, ..., a warp a tile. For a whole block.
// Blocks of zeros, whose scale is the lowest, do not count.
__device__ __forceinline__ int2 rangeOf(const MxMatrix& q, int matrix, int first, int step, int tiles, int chunks, int codeBytes)
{
    static_assert(TILE_WARPS == MX_RANGE_TILES, "");
    __shared__ int2 ofWarp[TILE_WARPS];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const unsigned char *scales = q.scales + static_cast<long long>(matrix) * tiles * MX_TILE_BYTES, *codes = q.codes + matrix * q.rows * codeBytes;
    uint32_t low = 255, high = 0, low4 = 0xffffffffu, high4 = 0;   // the latter: of four bytes each
    for (int tile = first + warp; tile < tiles; tile += step) {
        const uint4 u = *reinterpret_cast<const uint4*>(scales + static_cast<long long>(tile) * MX_TILE_BYTES + lane * 16);
        const uint32_t words[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((__vcmpeq4(words[i], 0) | __vcmpeq4(words[i], 0xffffffffu)) == 0) {
                low4 = __vminu4(low4, words[i]);
                high4 = __vmaxu4(high4, words[i]);
                continue;
            }
            const long long row = static_cast<long long>(tile / chunks) * MX_TILE + i * 32 + lane;
            for (int j = 0; j < 4; ++j) {
                const uint32_t scale = words[i] >> 8 * j & 255u;
                const int at = (tile % chunks * 4 + j) * 16;
                if (scale == 255) continue;   // (NaN, whatever it is divided by)
                if (scale == 0) {
                    if (row >= q.rows || at >= codeBytes) continue;
                    const uint4 c = *reinterpret_cast<const uint4*>(codes + row * codeBytes + at);
                    if (((c.x | c.y | c.z | c.w) & 0x77777777u) == 0) continue;
                }
                low = min(low, scale);
                high = max(high, scale);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        low = min(low, low4 >> 8 * j & 255u);
        high = max(high, high4 >> 8 * j & 255u);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) ofWarp[warp] = make_int2(static_cast<int>(low), static_cast<int>(high));
    __syncthreads();
    int2 all = ofWarp[0];
#pragma unroll
    for (int w = 1; w < TILE_WARPS; ++w) all = make_int2(min(all.x, ofWarp[w].x), max(all.y, ofWarp[w].y));
    return all;
}
__global__ void __launch_bounds__(TILE_THREADS) mx_ranges_kernel(const __grid_constant__ MxMatrix q, const __grid_constant__ MxWanted wanted, int2* __restrict__ found, int parts, int tiles,
                                                                 int chunks, int codeBytes)
{
    chained();
    const int matrix = blockIdx.x / parts, part = blockIdx.x - matrix * parts;
    if (!hasRows(wanted, matrix)) return;
    const int2 all = rangeOf(q, matrix, part * TILE_WARPS, parts * TILE_WARPS, tiles, chunks, codeBytes);
    if (threadIdx.x == 0) found[blockIdx.x] = all;
}
// What a matrix is divided by, 2^s, as 2^-s, for a whole block; written down (with whether its powers lie too far apart) by the block that has its first tile.
__device__ __forceinline__ float dividedBy(const MxMatrix& q, const MxRanges& ranges, unsigned matrix, bool first, int tiles, int chunks, int codeBytes)
{
    // Of a block in half: 0.5 * 2^-13 is its smallest normal number, 6 * 2^13 below its largest. Its subnormal ones reach down to -23, but a tensor core lines products up by their
    // operands' exponents, of which a subnormal one has the lowest whatever its bits are, and cuts off what lies 2^25 below the largest: sums of numbers 2^-9 below it lose as many bits.
    // (As they do from subnormal numbers of dy, in these products as in the 16-bit ones.)
    constexpr int LOWEST = 127 - 13, HIGHEST = 127 + 13;
    int low, high;
    if (ranges.parts == 0) {
        const int2 all = rangeOf(q, static_cast<int>(matrix), 0, TILE_WARPS, tiles, chunks, codeBytes);
        low = all.x;
        high = all.y;
    } else {
        const int lane = threadIdx.x & 31;
        const int2 f = lane < ranges.parts ? ranges.found[matrix * ranges.parts + lane] : make_int2(255, 0);
        low = __reduce_min_sync(0xffffffffu, f.x);
        high = __reduce_max_sync(0xffffffffu, f.y);
    }
    // (-114: the power and its inverse are normal numbers, and the lowest scale still is in reach)
    const int s = low >= LOWEST && high <= HIGHEST ? 0 : max(high - HIGHEST, -114);
    if (first && threadIdx.x == 0) {
        ranges.power[matrix] = powerOf(127 + s);
        ranges.apart[matrix] = low < LOWEST + s;
    }
    return powerOf(127 - s);
}

// Rows that 16-byte accesses cannot write: a warp per row, a lane per channel of a block, element by element side by side (20011 rows of 777 floats: 16 elements
// of a row per thread 75 us, so 20).
template <class T, int LANES, bool ALIGNED, bool DIVIDED>
__global__ void __launch_bounds__(TILE_THREADS) mx_dequantize_kernel(const __grid_constant__ MxMatrix q, T* __restrict__ y, long long stride, int tilesPerMatrix, int chunks,
                                                                     int codeBytes, const __grid_constant__ MxWanted wanted, const __grid_constant__ MxRanges ranges)
{
    chained();
    const unsigned tile = blockIdx.x / static_cast<unsigned>(chunks);
    const int chunk = static_cast<int>(blockIdx.x - tile * chunks);
    const RowTile t = rowTile(q, tilesPerMatrix, tile);
    const unsigned matrix = tile / static_cast<unsigned>(tilesPerMatrix);
    const bool first = chunk == 0 && tile == matrix * tilesPerMatrix;
    if (!hasRows(wanted, matrix)) {
        if (DIVIDED && first && threadIdx.x == 0) {
            ranges.power[matrix] = 1.f;
            ranges.apart[matrix] = 0;
        }
        return;
    }
    float down = 1.f;
    if constexpr (DIVIDED) down = dividedBy(q, ranges, matrix, first, tilesPerMatrix * chunks, chunks, codeBytes);
    const unsigned char *codes = q.codes + t.row * codeBytes, *scales = q.scales + static_cast<long long>(blockIdx.x) * MX_TILE_BYTES;
    if constexpr (!ALIGNED) {
        constexpr int AT_ONCE = 4, BLOCKS = MX_TILE / MX_BLOCK;
        const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, c = chunk * MX_TILE + lane, shift = (lane & 1) * 4;
        int at[BLOCKS];   // of a lane's code in a row
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) at[b] = min(c + b * MX_BLOCK, q.channels - 1) / 2;
        for (int i = warp; i < t.rows; i += TILE_WARPS * AT_ONCE) {
            uint32_t code[AT_ONCE][BLOCKS], scale[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int r = min(i + k * TILE_WARPS, t.rows - 1);
                const unsigned char* row = codes + static_cast<long long>(r) * codeBytes;
                scale[k] = scales[(r & 31) * 16 + (r >> 5) * 4 + (lane & 3)];   // a lane per block
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) code[k][b] = row[at[b]];
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int r = i + k * TILE_WARPS;
                if (r >= t.rows) break;
                const float power = powerOf(scale[k]) * down;
                T* row = y + (t.row + r) * stride + c;
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
                    const float v = decodeOne(code[k][b] >> shift) * __shfl_sync(0xffffffffu, power, b);
                    if (c + b * MX_BLOCK < q.channels) row[b * MX_BLOCK] = Element<T>::from(v);
                }
            }
        }
    } else {
        // 16 bytes of a row a thread, neighbours side by side
        constexpr int W = WIDE<T>, ROW = LANES * SIXTEEN / W, STEP = TILE_THREADS / ROW, PASSES = MX_TILE / STEP, AT_ONCE = PASSES < 8 ? PASSES : 8;
        const int lane = threadIdx.x % ROW, first = threadIdx.x / ROW, c = chunk * MX_TILE + lane * W;
        if (c >= q.channels) return;
        codes += c / 2;
        T* at = y + (t.row + first) * stride + c;
#pragma unroll
        for (int begin = 0; begin < PASSES; begin += AT_ONCE) {
            uint32_t code[AT_ONCE], scale[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int r = min((begin + i) * STEP + first, t.rows - 1);
                if constexpr (W == 8) code[i] = *reinterpret_cast<const uint32_t*>(codes + static_cast<long long>(r) * codeBytes);
                else code[i] = *reinterpret_cast<const uint16_t*>(codes + static_cast<long long>(r) * codeBytes);
                scale[i] = scales[(r & 31) * 16 + (r >> 5) * 4 + lane * W / MX_BLOCK];
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                float f[8], out[W];
                if constexpr (W == 8) decodeEight(code[i], f);
                else {
#pragma unroll
                    for (int j = 0; j < W; ++j) f[j] = decodeOne(code[i] >> 4 * j);
                }
                const float power = powerOf(scale[i]) * down;
#pragma unroll
                for (int j = 0; j < W; ++j) out[j] = f[j] * power;
                if ((begin + i) * STEP + first < t.rows) store<T, W>(at, pack<T, W>(out));
                at += STEP * stride;
            }
        }
    }
}

template <class T>
cudaError_t quantize(const MxMatrix& q, int type, const Rows& x, unsigned blocks, cudaStream_t stream)
{
    return byLanes(x, type, q.channels, [&](auto lanes, auto aligned) {
        launchChained(mx_quantize_kernel<T, decltype(lanes)::value, decltype(aligned)::value>, blocks, TILE_THREADS, 0, stream, 1, q, static_cast<const T*>(x.data), x.stride, mxTiles(q.rows),
                      mxTiles(q.channels), mxCodeBytes(q.channels));
        return cudaGetLastError();
    });
}
template <class T, bool DIVIDED = false>
cudaError_t dequantize(const MxMatrix& q, int type, const Rows& y, unsigned blocks, cudaStream_t stream, const MxWanted& wanted, const MxRanges& ranges = {})
{
    return byLanes(y, type, wanted.padded ? (q.channels + 7) / 8 * 8 : q.channels, [&](auto lanes, auto aligned) {
        launchChained(mx_dequantize_kernel<T, decltype(aligned)::value ? decltype(lanes)::value : 8, decltype(aligned)::value, DIVIDED>, blocks, TILE_THREADS, 0, stream, 1, q,
                      static_cast<T*>(y.data), y.stride, mxTiles(q.rows), mxTiles(q.channels), mxCodeBytes(q.channels), wanted, ranges);
        return cudaGetLastError();
    });
}
bool blocksOf(const MxMatrix& q, unsigned& blocks)
{
    const long long n = q.matrices * mxTiles(q.rows) * mxTiles(q.channels);
    blocks = static_cast<unsigned>(n);
    return n <= 0x7fffffff;
}

} // namespace

cudaError_t launchMxQuantize(const MxMatrix& q, int type, const Rows& x, cudaStream_t stream)
{
    unsigned blocks;
    if (!blocksOf(q, blocks)) return cudaErrorInvalidConfiguration;
    if (blocks == 0) return cudaSuccess;
    return type == TYPE_FLOAT ? quantize<float>(q, type, x, blocks, stream) : type == TYPE_HALF ? quantize<__half>(q, type, x, blocks, stream) : quantize<__nv_bfloat16>(q, type, x, blocks, stream);
}
cudaError_t launchMxRanges(const MxMatrix& q, const MxWanted& wanted, const MxRanges& ranges, cudaStream_t stream)
{
    if (ranges.parts == 0) return cudaSuccess;
    const int chunks = mxTiles(q.channels);
    launchChained(mx_ranges_kernel, static_cast<unsigned>(q.matrices * ranges.parts), TILE_THREADS, 0, stream, 1, q, wanted, ranges.found, ranges.parts, mxTiles(q.rows) * chunks, chunks,
                  mxCodeBytes(q.channels));
    return cudaGetLastError();
}
cudaError_t launchMxDequantize(const MxMatrix& q, int type, const Rows& y, cudaStream_t stream, const MxWanted& wanted, const MxRanges* ranges)
{
    unsigned blocks;
    if (!blocksOf(q, blocks)) return cudaErrorInvalidConfiguration;
    if (blocks == 0) return cudaSuccess;
    if (ranges != nullptr && type != TYPE_HALF) return cudaErrorInvalidValue;
    if (ranges != nullptr) return dequantize<__half, true>(q, type, y, blocks, stream, wanted, *ranges);
    return type == TYPE_FLOAT ? dequantize<float>(q, type, y, blocks, stream, wanted) : type == TYPE_HALF ? dequantize<__half>(q, type, y, blocks, stream, wanted) : dequantize<__nv_bfloat16>(q, type, y, blocks, stream, wanted);
}

} // namespace kernel
} // namespace qmlp
