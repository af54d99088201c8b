// Launchers of the operators on feature rows: layer norm, embedding lookup, routing to experts, products grouped by expert, dropout, 4-bit matrices
// and their products.
// The arguments are checked by the entry points (capi_operators.cpp); every launcher returns the status of its launches.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace qmlp {
namespace kernel {

// element types, numbered as the precisions of the C ABI
enum : int { TYPE_FLOAT = 0, TYPE_HALF = 1, TYPE_BFLOAT16 = 3, TYPE_INT32 = 4, TYPE_INT64 = 5 };
inline int typeBytes(int type) { return type == TYPE_FLOAT || type == TYPE_INT32 ? 4 : type == TYPE_INT64 ? 8 : 2; }

// rows of `channels` consecutive elements, `stride` elements apart
struct Rows {
    void* data;
    long long stride;
};
// optional vector of `channels` elements of type `type`
struct Vector {
    const void* data;
    int type;
};

// ---- layer norm ------------------------------------------------------------------------------------------------------
struct LayerNormArgs {
    long long rows;
    int channels, type, numSMs;
    float epsilon;
    Rows x, y;            // input, output
    Vector weight, bias;
    float* stats;         // rows means, then rows reciprocal deviations; may be null in the forward pass
    // adjoint
    Rows gradY, gradX;    // gradX.data may be null
    void *gradWeight, *gradBias;   // of type weight.type / gradBiasType, may be null
    int gradWeightType, gradBiasType;
    float* partial;       // scratch: layerNormPartials() rows of 2 x channels sums
    int* status;          // the library's status word
    int ringStages;       // set by the launcher
};
// blocks whose partial sums of the parameters' gradients the adjoint leaves in its scratch (an upper bound)
int layerNormPartials(long long rows, int channels, int type, int numSMs);
cudaError_t launchLayerNormForward(const LayerNormArgs& a, cudaStream_t stream);
cudaError_t launchLayerNormAdjoint(const LayerNormArgs& a, cudaStream_t stream);

// ---- embedding lookup ------------------------------------------------------------------------------------------------
struct EmbeddingArgs {
    long long tokens, rows;
    int channels, type, tokenType, numSMs;
    float scale;
    const void* token;
    long long tokenStride;
    Rows table, y;
    // adjoint
    Rows gradY, gradTable;
    void* scratch;
};
size_t embeddingAdjointBytes(long long tokens, long long rows, int channels, int type, int numSMs);
cudaError_t launchEmbeddingForward(const EmbeddingArgs& a, cudaStream_t stream);
cudaError_t launchEmbeddingAdjoint(const EmbeddingArgs& a, cudaStream_t stream);

// ---- routing -----------------------------------------------------------------------------------------------------------
constexpr int ROUTE_MAX_EXPERTS = 1024, ROUTE_MAX_CHOSEN = 32;
struct RouteArgs {
    long long tokens;
    int experts, chosen, type, normalize;
    Rows logits;
    float* weights;       // (tokens, chosen)
    int *expert, *order, *position, *offsets;
    void* scratch;
    // adjoint
    const float* gradWeights;
    Rows gradLogits;
};
size_t routeBytes(long long tokens, int experts, int chosen);
cudaError_t launchRouteForward(const RouteArgs& a, cudaStream_t stream);
cudaError_t launchRouteAdjoint(const RouteArgs& a, cudaStream_t stream);

struct ExchangeArgs {
    long long tokens;
    int chosen, channels, type, numSMs;
    Rows x, rows;              // (tokens, channels), (tokens * chosen, channels)
    const int *order, *position;
    const float* weights;      // (tokens, chosen)
    Rows gradX, gradRows;      // gradRows.data may be null
    float* gradWeights;        // may be null
};
cudaError_t launchDispatch(const ExchangeArgs& a, cudaStream_t stream);         // x -> rows
cudaError_t launchDispatchAdjoint(const ExchangeArgs& a, cudaStream_t stream);  // gradRows -> gradX
cudaError_t launchCombine(const ExchangeArgs& a, cudaStream_t stream);          // rows -> x
cudaError_t launchCombineAdjoint(const ExchangeArgs& a, cudaStream_t stream);   // gradX, rows -> gradRows, gradWeights

// ---- products grouped by expert ------------------------------------------------------------------------------------------
constexpr int EXPERTS_MAX = 2048;
struct ExpertArgs {
    long long rows;
    int experts, channelsIn, channelsOut, type, numSMs;
    Rows x, y;
    const void* weight;        // (experts, channelsOut, channelsIn), contiguous
    const void* bias;          // (experts, channelsOut), contiguous, may be null
    const int* offsets;        // experts + 1
    // adjoint
    Rows gradY, gradX;         // gradX.data may be null
    void *gradWeight, *gradBias;   // may be null
    void* scratch;
    int* status;
    // column sums of gradY beside an input gradient alone (null: none): expertSums rows of channelsOut floats, expertSumsPerUnit for every unit of rows of an
    // expert, one expert's behind another's; units of the experts in front of each (experts + 1)
    float* columnSums;
    int* unitsBefore;
    const float* powers;   // of each expert, what its rows of an input gradient alone are multiplied with before they are rounded (null: one)
    int weightStride;      // adjoint: elements between rows of weight (0: channelsIn)
};
int expertSumsPerUnit(const ExpertArgs& a);
long long expertSums(const ExpertArgs& a);   // an upper bound
// scratch of a forward call (adjoint = false) or an adjoint call
size_t expertBytes(const ExpertArgs& a, bool adjoint);
cudaError_t launchExpertForward(const ExpertArgs& a, cudaStream_t stream);
cudaError_t launchExpertAdjoint(const ExpertArgs& a, cudaStream_t stream);

// ---- dropout ---------------------------------------------------------------------------------------------------------------
struct DropoutArgs {
    long long rows;
    int channels, type;
    Rows x, residual, y;       // residual.data may be null
    unsigned cut;              // of 65536 numbers, those below it drop
    unsigned long long seed, offset;
    const long long* step;     // added to the offset, may be null
};
cudaError_t launchDropout(const DropoutArgs& a, cudaStream_t stream);

// ---- microscaled 4-bit matrices ----------------------------------------------------------------------------------------------
// `matrices` matrices of (rows, channels). Codes: rows of mxCodeBytes(channels), two e2m1 elements a byte, the first in the low bits, zeros behind the
// last channel. Scales: tiles of 128 rows x 128 channels, 512 bytes each, [matrix][row tile][channel tile]; the exponent (+ 127) of row 32 q + i and of
// the channels from 32 j on lies at byte 16 i + 4 q + j of its tile, where a tensor core's scales come from without a change.
constexpr int MX_BLOCK = 32, MX_TILE = 128, MX_TILE_BYTES = 512;
inline int mxBlocks(int channels) { return (channels + MX_BLOCK - 1) / MX_BLOCK; }
inline int mxCodeBytes(int channels) { return mxBlocks(channels) * (MX_BLOCK / 2); }
inline int mxTiles(long long n) { return static_cast<int>((n + MX_TILE - 1) / MX_TILE); }
struct MxMatrix {
    long long matrices, rows;
    int channels;
    unsigned char *codes, *scales;
};
cudaError_t launchMxQuantize(const MxMatrix& q, int type, const Rows& x, cudaStream_t stream);
// How far the powers of two of each matrix reach. Half has the elements (0.5 to 6) of 27 neighbouring powers of two as normal numbers, its
// own being -13 to 13: a matrix that leaves it is divided by a power of two, `power`, so that its largest numbers come to the upper end; `apart`: its powers
// lie farther apart than half holds. found: the lowest and highest power (+ 127) that a `parts`-th of a matrix has; (255, 0) for none.
struct MxRanges {
    int parts;
    int2* found;     // matrices x parts
    float* power;    // matrices; written with the decoded matrices, as
    int* apart;      // matrices
};
// most parts of a matrix; tiles of scales that a block takes at once, which is where "small" ends (8 experts of 64 x 64 half: 6.0 us for ranges and decoding, so 4.5; 32 of 300 x 777, 21
// tiles: 18.0 us, 21.1 if every block read them all)
constexpr int MX_RANGE_PARTS = 32, MX_RANGE_TILES = 8;
inline int mxRangeParts(const MxMatrix& q)
{
    const long long n = (static_cast<long long>(mxTiles(q.rows)) * mxTiles(q.channels) + MX_RANGE_TILES - 1) / MX_RANGE_TILES;
    return n <= 1 ? 0 : n < MX_RANGE_PARTS ? static_cast<int>(n) : MX_RANGE_PARTS;
}
// Of matrices of experts, those that are wanted: of experts that have rows, or all (offsets null). (Gradient of 2 rows of 64 experts of 1024 -> 2048 bfloat16: all
// matrices decoded 75 us, those of the two 27 us.)
struct MxWanted {
    const int* offsets;   // matrices + 1
    long long rows;
    bool padded;          // of 16-bit y: what lies behind a row up to a multiple of 8 channels may be written (zeros)
};
cudaError_t launchMxRanges(const MxMatrix& q, const MxWanted& wanted, const MxRanges& ranges, cudaStream_t stream);
// `ranges`: of half y, whose matrices are divided by their powers; null: as they are
cudaError_t launchMxDequantize(const MxMatrix& q, int type, const Rows& y, cudaStream_t stream, const MxWanted& wanted = {}, const MxRanges* ranges = nullptr);

// products of rows with such matrices (weight.matrices experts, weight.rows channels out)
struct MxLinearArgs {
    long long rows;
    int type, numSMs;
    Rows x, y;
    MxMatrix weight;
    const void* bias;          // (experts, channels out), contiguous, may be null
    const int* offsets;        // experts + 1; null: all rows are the one expert's
    // adjoint
    Rows gradY, gradX;         // gradX.data may be null
    void* gradBias;            // may be null
    void* scratch;
    int* status;
};
size_t mxLinearBytes(const MxLinearArgs& a);
size_t mxLinearAdjointBytes(const MxLinearArgs& a);
cudaError_t launchMxLinear(const MxLinearArgs& a, cudaStream_t stream);
cudaError_t launchMxLinearAdjoint(const MxLinearArgs& a, cudaStream_t stream);

} // namespace kernel
} // namespace qmlp
