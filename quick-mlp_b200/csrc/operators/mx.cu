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
__device__ __forceinline__ RowTile rowTile(const MxMatrix& q, int tilesPerMatrix, long long tile)
{
    const long long matrix = tile / tilesPerMatrix, within = (tile - matrix * tilesPerMatrix) * MX_TILE;
    return {matrix * q.rows + within, static_cast<int>(min(static_cast<long long>(MX_TILE), q.rows - within))};
}

template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_quantize_kernel(const __grid_constant__ MxMatrix q, const T* __restrict__ x, long long stride, int tilesPerMatrix, int chunks,
                                                                   int codeBytes)
{
    chained();
    __shared__ uint4 words[MX_TILE / 4];
    const long long tile = blockIdx.x / chunks;
    const int chunk = blockIdx.x - static_cast<int>(tile) * chunks;
    const RowTile t = rowTile(q, tilesPerMatrix, tile);
    quantizeTile<T, LANES, ALIGNED>(x + t.row * stride, stride, t.rows, chunk, q.channels, q.codes + t.row * codeBytes, codeBytes,
                                    q.scales + (tile * chunks + chunk) * MX_TILE_BYTES, reinterpret_cast<uint32_t*>(words));
}

template <class T, int LANES, bool ALIGNED>
__global__ void __launch_bounds__(TILE_THREADS) mx_dequantize_kernel(const __grid_constant__ MxMatrix q, T* __restrict__ y, long long stride, int tilesPerMatrix, int chunks,
                                                                     int codeBytes)
{
    chained();
    constexpr int PASSES = TILE_PASSES<LANES>, STEP = TILE_THREADS / LANES;
    const long long tile = blockIdx.x / chunks;
    const int chunk = blockIdx.x - static_cast<int>(tile) * chunks;
    const RowTile t = rowTile(q, tilesPerMatrix, tile);
    const int lane = threadIdx.x % LANES, first = threadIdx.x / LANES, c = chunk * MX_TILE + lane * 8;
    if (c >= q.channels) return;
    const unsigned char *codes = q.codes + t.row * codeBytes + c / 2, *scales = q.scales + (tile * chunks + chunk) * MX_TILE_BYTES + lane / 4;
    uint32_t code[PASSES], scale[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * STEP + first;
        code[i] = scale[i] = 0;
        if (r >= t.rows) continue;
        code[i] = *reinterpret_cast<const uint32_t*>(codes + static_cast<long long>(r) * codeBytes);
        scale[i] = scales[(r & 31) * 16 + (r >> 5) * 4];
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * STEP + first;
        if (r >= t.rows) break;
        float f[8];
        decodeEight(code[i], f);
        const float power = powerOf(scale[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= power;
        T* at = y + (t.row + r) * stride + c;
        if constexpr (ALIGNED) {
#pragma unroll
            for (int k = 0; k < 8 / WIDE<T>; ++k) store<T, WIDE<T>>(at + k * WIDE<T>, pack<T, WIDE<T>>(*reinterpret_cast<const float (*)[WIDE<T>]>(&f[k * WIDE<T>])));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < q.channels) at[j] = Element<T>::from(f[j]);
        }
    }
}

// whether rows allow accesses of eight elements
template <class T>
bool aligned(const Rows& r, int channels)
{
    return (reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.stride % WIDE<T> == 0 && channels % 8 == 0;
}
// calls f(lanes, aligned) with both as constants
template <class F>
cudaError_t byShape(int channels, bool aligned, F&& f)
{
    auto lanes = [&](auto n) { return aligned ? f(n, std::true_type()) : f(n, std::false_type()); };
    switch (lanesOf(channels)) {
    case 4: return lanes(std::integral_constant<int, 4>());
    case 8: return lanes(std::integral_constant<int, 8>());
    default: return lanes(std::integral_constant<int, 16>());
    }
}
template <class T>
cudaError_t quantize(const MxMatrix& q, const Rows& x, unsigned blocks, cudaStream_t stream)
{
    return byShape(q.channels, aligned<T>(x, q.channels), [&](auto lanes, auto whole) {
        launchChained(mx_quantize_kernel<T, decltype(lanes)::value, decltype(whole)::value>, blocks, TILE_THREADS, 0, stream, 1, q, static_cast<const T*>(x.data), x.stride,
                      mxTiles(q.rows), mxTiles(q.channels), mxCodeBytes(q.channels));
        return cudaGetLastError();
    });
}
template <class T>
cudaError_t dequantize(const MxMatrix& q, const Rows& y, unsigned blocks, cudaStream_t stream)
{
    return byShape(q.channels, aligned<T>(y, q.channels), [&](auto lanes, auto whole) {
        launchChained(mx_dequantize_kernel<T, decltype(lanes)::value, decltype(whole)::value>, blocks, TILE_THREADS, 0, stream, 1, q, static_cast<T*>(y.data), y.stride,
                      mxTiles(q.rows), mxTiles(q.channels), mxCodeBytes(q.channels));
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
    return type == TYPE_FLOAT ? quantize<float>(q, x, blocks, stream) : type == TYPE_HALF ? quantize<__half>(q, x, blocks, stream) : quantize<__nv_bfloat16>(q, x, blocks, stream);
}
cudaError_t launchMxDequantize(const MxMatrix& q, int type, const Rows& y, cudaStream_t stream)
{
    unsigned blocks;
    if (!blocksOf(q, blocks)) return cudaErrorInvalidConfiguration;
    if (blocks == 0) return cudaSuccess;
    return type == TYPE_FLOAT ? dequantize<float>(q, y, blocks, stream) : type == TYPE_HALF ? dequantize<__half>(q, y, blocks, stream) : dequantize<__nv_bfloat16>(q, y, blocks, stream);
}

} // namespace kernel
} // namespace qmlp
