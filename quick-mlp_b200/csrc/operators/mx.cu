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

// Rows that 16-byte accesses cannot write: a warp per row, a lane per channel of a block, element by element side by side (20011 rows of 777 floats: 16 elements
// of a row per thread 75 us, so 20).
template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_dequantize_kernel(const __grid_constant__ MxMatrix q, T* __restrict__ y, long long stride, int tilesPerMatrix, int chunks,
                                                                     int codeBytes)
{
    chained();
    const unsigned tile = blockIdx.x / static_cast<unsigned>(chunks);
    const int chunk = static_cast<int>(blockIdx.x - tile * chunks);
    const RowTile t = rowTile(q, tilesPerMatrix, tile);
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
                const float power = powerOf(scale[k]);
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
                const float power = powerOf(scale[i]);
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
template <class T>
cudaError_t dequantize(const MxMatrix& q, int type, const Rows& y, unsigned blocks, cudaStream_t stream)
{
    return byLanes(y, type, q.channels, [&](auto lanes, auto aligned) {
        launchChained(mx_dequantize_kernel<T, decltype(aligned)::value ? decltype(lanes)::value : 8, decltype(aligned)::value>, blocks, TILE_THREADS, 0, stream, 1, q, static_cast<T*>(y.data), y.stride, mxTiles(q.rows),
                      mxTiles(q.channels), mxCodeBytes(q.channels));
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
cudaError_t launchMxDequantize(const MxMatrix& q, int type, const Rows& y, cudaStream_t stream)
{
    unsigned blocks;
    if (!blocksOf(q, blocks)) return cudaErrorInvalidConfiguration;
    if (blocks == 0) return cudaSuccess;
    return type == TYPE_FLOAT ? dequantize<float>(q, type, y, blocks, stream) : type == TYPE_HALF ? dequantize<__half>(q, type, y, blocks, stream) : dequantize<__nv_bfloat16>(q, type, y, blocks, stream);
}

} // namespace kernel
} // namespace qmlp
