// Launchers of the operators on feature rows: layer norm, embedding lookup, routing to experts, products grouped by expert.
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
};
// scratch of a forward call (adjoint = false) or an adjoint call
size_t expertBytes(const ExpertArgs& a, bool adjoint);
cudaError_t launchExpertForward(const ExpertArgs& a, cudaStream_t stream);
cudaError_t launchExpertAdjoint(const ExpertArgs& a, cudaStream_t stream);

} // namespace kernel
} // namespace qmlp
