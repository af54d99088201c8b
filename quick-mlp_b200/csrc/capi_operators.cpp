// extern "C" entry points of the operators on feature rows: layer norm, embedding lookup, routing to experts, products grouped
// by expert, dropout, 4-bit matrices and their products. No counterpart in the reference: its callers write them in PyTorch around the network.
#include "entry.hpp"
#include "operators/operators.h"

#include <cmath>

using namespace qmlp;

namespace {

// records of qmlp_read_kernel_timing: one per call of an operator
enum : int {
    KERNEL_ID_LAYER_NORM_FORWARD = 110, KERNEL_ID_LAYER_NORM_ADJOINT, KERNEL_ID_EMBEDDING_FORWARD, KERNEL_ID_EMBEDDING_ADJOINT, KERNEL_ID_ROUTE_FORWARD,
    KERNEL_ID_ROUTE_ADJOINT, KERNEL_ID_DISPATCH_FORWARD, KERNEL_ID_DISPATCH_ADJOINT, KERNEL_ID_COMBINE_FORWARD, KERNEL_ID_COMBINE_ADJOINT,
    KERNEL_ID_EXPERT_LINEAR_FORWARD, KERNEL_ID_EXPERT_LINEAR_ADJOINT, KERNEL_ID_DROPOUT, KERNEL_ID_MX_QUANTIZE, KERNEL_ID_MX_DEQUANTIZE, KERNEL_ID_MX_LINEAR_FORWARD,
    KERNEL_ID_MX_LINEAR_ADJOINT
};
constexpr int64_t MAX_CHANNELS = 1 << 20, MAX_ROWS = (1ll << 31) - 4096, MAX_SORTED = 1ll << 30;

template <class F>
int launch(int id, qmlp_stream_t stream, F&& f)
{
    TimedLaunch timed(id, static_cast<cudaStream_t>(stream));
    checkCuda(f(static_cast<cudaStream_t>(stream)), "kernel launch failed");
    return QMLP_OK;
}

bool defined(const qmlp_tensor_t* t) { return t != nullptr && t->ndim > 0; }

// a matrix of features: float, half or bfloat16, the elements of a row side by side
void checkFeatures(const qmlp_tensor_t* t, const char* name, bool written)
{
    checkDim(t, 2, name);
    if (t->precision != QMLP_FLOAT && t->precision != QMLP_HALF && t->precision != QMLP_BFLOAT16)
        throw std::runtime_error(format("%s has the wrong data type, expected float, half or bfloat16", name));
    if (t->sizes[0] < 0 || t->sizes[0] > MAX_ROWS) throw std::runtime_error(format("%s has too many rows (%lld)", name, static_cast<long long>(t->sizes[0])));
    if (t->sizes[1] < 1 || t->sizes[1] > MAX_CHANNELS)
        throw std::runtime_error(format("%s must have 1 to %lld channels, got %lld", name, static_cast<long long>(MAX_CHANNELS), static_cast<long long>(t->sizes[1])));
    if (t->sizes[1] > 1 && t->sizes[0] > 0 && t->strides[1] != 1) throw std::runtime_error(format("the elements of a row of %s must lie side by side (stride 1)", name));
    if (t->sizes[0] > 1 && (t->strides[0] < 0 || (written && t->strides[0] < t->sizes[1]))) throw std::runtime_error(format("the rows of %s overlap", name));
}
void checkLike(const qmlp_tensor_t* t, const qmlp_tensor_t* like, const char* name, bool written)
{
    checkFeatures(t, name, written);
    checkDtype(t, like->precision, name);
    checkSize(t, 0, like->sizes[0], name);
    checkSize(t, 1, like->sizes[1], name);
}
// rows with a row stride that is valid for a single row too
kernel::Rows rowsOf(const qmlp_tensor_t* t) { return {t->data, t->sizes[0] > 1 ? t->strides[0] : t->sizes[1]}; }
// parameters of a layer: a contiguous vector of float32 or of the features' type
kernel::Vector vectorOf(const qmlp_tensor_t* t, const qmlp_tensor_t* features, const char* name)
{
    if (!defined(t)) return {nullptr, 0};
    checkDim(t, 1, name);
    checkSize(t, 0, features->sizes[1], name);
    if (t->precision != QMLP_FLOAT && t->precision != features->precision)
        throw std::runtime_error(format("%s has the wrong data type, expected float or %s", name, precisionName(features->precision)));
    if (t->sizes[0] > 1 && t->strides[0] != 1) throw std::runtime_error(format("%s must be contiguous", name));
    return {t->data, t->precision};
}
void checkScratch(const void* memory, size_t given, size_t needed)
{
    if (needed == 0) return;
    if (memory == nullptr || given < needed)
        throw std::runtime_error(format("scratch memory of %llu bytes is needed, got %llu", static_cast<unsigned long long>(needed),
                                        static_cast<unsigned long long>(memory == nullptr ? 0 : given)));
    if ((reinterpret_cast<uintptr_t>(memory) & 255) != 0) throw std::runtime_error("scratch memory must be 256-byte aligned");
}
void checkPointer(const void* p, const char* name)
{
    if (p == nullptr) throw std::runtime_error(std::string(name) + " is undefined");
}

kernel::LayerNormArgs layerNorm(const qmlp_tensor_t* input)
{
    kernel::LayerNormArgs a{};
    a.rows = input->sizes[0];
    a.channels = static_cast<int>(input->sizes[1]);
    a.type = input->precision;
    a.x = rowsOf(input);
    return a;
}
size_t layerNormAdjointBytes(int64_t rows, int channels, int precision)
{
    return rows == 0 ? 0 : static_cast<size_t>(kernel::layerNormPartials(rows, channels, precision, Library::instance().smCount())) * 2 * channels * sizeof(float);
}

void checkTokens(const qmlp_tensor_t* t)
{
    checkDim(t, 1, "tokens");
    if (t->precision != QMLP_INT32 && t->precision != QMLP_INT64) throw std::runtime_error("tokens has the wrong data type, expected int32 or int64");
    if (t->sizes[0] > MAX_ROWS) throw std::runtime_error(format("tokens has too many entries (%lld)", static_cast<long long>(t->sizes[0])));
}

void checkRouting(const qmlp_routing_t* r)
{
    if (r == nullptr) throw std::runtime_error("routing is undefined");
    if (r->num_experts < 1 || r->num_experts > kernel::ROUTE_MAX_EXPERTS)
        throw std::runtime_error(format("a router has 1 to %d experts, got %d", kernel::ROUTE_MAX_EXPERTS, r->num_experts));
    if (r->chosen < 1 || r->chosen > kernel::ROUTE_MAX_CHOSEN || r->chosen > r->num_experts)
        throw std::runtime_error(format("a row chooses 1 to %d of its experts, got %d of %d", kernel::ROUTE_MAX_CHOSEN, r->chosen, r->num_experts));
    if (r->tokens < 0 || r->tokens > MAX_ROWS / r->chosen) throw std::runtime_error(format("too many rows to route (%lld)", static_cast<long long>(r->tokens)));
}
kernel::ExchangeArgs exchange(const qmlp_routing_t* r, const qmlp_tensor_t* features)
{
    checkRouting(r);
    kernel::ExchangeArgs a{};
    a.tokens = r->tokens;
    a.chosen = r->chosen;
    a.channels = static_cast<int>(features->sizes[1]);
    a.type = features->precision;
    a.order = r->order;
    a.position = r->positions;
    a.weights = r->weights;
    a.numSMs = Library::instance().smCount();
    return a;
}
void checkSlots(const qmlp_tensor_t* t, const qmlp_routing_t* r, const qmlp_tensor_t* features, const char* name, bool written)
{
    checkFeatures(t, name, written);
    checkDtype(t, features->precision, name);
    checkSize(t, 0, r->tokens * r->chosen, name);
    checkSize(t, 1, features->sizes[1], name);
}

kernel::ExpertArgs experts(const qmlp_tensor_t* input, const qmlp_tensor_t* weight, int num_experts)
{
    checkFeatures(input, "input", false);
    if (input->precision == QMLP_FLOAT) throw std::runtime_error("input has the wrong data type, expected half or bfloat16");
    if (num_experts < 1 || num_experts > kernel::EXPERTS_MAX) throw std::runtime_error(format("1 to %d experts are supported, got %d", kernel::EXPERTS_MAX, num_experts));
    checkFeatures(weight, "weight", false);
    checkDtype(weight, input->precision, "weight");
    checkSize(weight, 1, input->sizes[1], "weight");
    if (weight->sizes[0] < num_experts || weight->sizes[0] % num_experts != 0 || weight->sizes[0] / num_experts > MAX_CHANNELS)
        throw std::runtime_error(format("weight must have the channels out of %d experts as rows, got %lld", num_experts, static_cast<long long>(weight->sizes[0])));
    if (weight->sizes[0] > 1 && weight->strides[0] != weight->sizes[1]) throw std::runtime_error("weight must be contiguous");
    kernel::ExpertArgs a{};
    a.rows = input->sizes[0];
    a.experts = num_experts;
    a.channelsIn = static_cast<int>(input->sizes[1]);
    a.channelsOut = static_cast<int>(weight->sizes[0] / num_experts);
    a.type = input->precision;
    a.x = rowsOf(input);
    a.weight = weight->data;
    return a;
}
const void* expertBias(const qmlp_tensor_t* bias, const kernel::ExpertArgs& a, const char* name)
{
    if (!defined(bias)) return nullptr;
    checkDim(bias, 2, name);
    checkDtype(bias, a.type, name);
    checkSize(bias, 0, a.experts, name);
    checkSize(bias, 1, a.channelsOut, name);
    if ((a.channelsOut > 1 && bias->strides[1] != 1) || (a.experts > 1 && bias->strides[0] != a.channelsOut)) throw std::runtime_error(format("%s must be contiguous", name));
    return bias->data;
}
void expertGradients(kernel::ExpertArgs& a, const qmlp_tensor_t* adjOutput, const qmlp_tensor_t* input)
{
    checkFeatures(adjOutput, "adj_output", false);
    checkDtype(adjOutput, a.type, "adj_output");
    checkSize(adjOutput, 0, input->sizes[0], "adj_output");
    checkSize(adjOutput, 1, a.channelsOut, "adj_output");
    a.gradY = rowsOf(adjOutput);
}

void checkMx(const qmlp_mx_t* m, const char* name)
{
    if (m == nullptr) throw std::runtime_error(std::string(name) + " is undefined");
    if (m->channels < 1 || m->channels > MAX_CHANNELS)
        throw std::runtime_error(format("%s must have 1 to %lld channels, got %d", name, static_cast<long long>(MAX_CHANNELS), m->channels));
    if (m->matrices < 0 || m->rows < 0 || m->matrices > MAX_ROWS || (m->matrices > 0 && m->rows > MAX_ROWS / m->matrices)) throw std::runtime_error(format("%s has too many rows", name));
    if (m->matrices * kernel::mxTiles(m->rows) > 0x7fffffffll / kernel::mxTiles(m->channels)) throw std::runtime_error(format("%s has too many tiles of scales", name));
    if (m->matrices == 0 || m->rows == 0) return;
    if (m->codes == nullptr || m->scales == nullptr) throw std::runtime_error(std::string(name) + " is undefined");
    if (((reinterpret_cast<uintptr_t>(m->codes) | reinterpret_cast<uintptr_t>(m->scales)) & 15) != 0) throw std::runtime_error(format("the arrays of %s must be 16-byte aligned", name));
}
kernel::MxMatrix matrixOf(const qmlp_mx_t* m) { return {m->matrices, m->rows, m->channels, m->codes, m->scales}; }
void checkMxFeatures(const qmlp_tensor_t* t, const qmlp_mx_t* m, const char* name, bool written)
{
    checkFeatures(t, name, written);
    checkSize(t, 0, m->matrices * m->rows, name);
    checkSize(t, 1, m->channels, name);
}
// products with 4-bit matrices of the rows of `rows`, which have `channels` channels
kernel::MxLinearArgs mxLinear(const qmlp_tensor_t* rows, const qmlp_mx_t* weight, int64_t channels, const char* name)
{
    checkFeatures(rows, name, false);
    if (rows->precision == QMLP_FLOAT) throw std::runtime_error(format("%s has the wrong data type, expected half or bfloat16", name));
    checkMx(weight, "weight");
    if (weight->matrices < 1 || weight->matrices > kernel::EXPERTS_MAX)
        throw std::runtime_error(format("1 to %d experts are supported, got %lld", kernel::EXPERTS_MAX, static_cast<long long>(weight->matrices)));
    if (weight->rows < 1 || weight->rows > MAX_CHANNELS)
        throw std::runtime_error(format("weight must have 1 to %lld channels out, got %lld", static_cast<long long>(MAX_CHANNELS), static_cast<long long>(weight->rows)));
    checkSize(rows, 1, channels, name);
    kernel::MxLinearArgs a{};
    a.rows = rows->sizes[0];
    // (two tiles of 128 rows per expert may be partly empty)
    if (a.rows / kernel::MX_TILE + 2 * kernel::EXPERTS_MAX > 0x7fffffffll / kernel::mxTiles(weight->channels))
        throw std::runtime_error(format("%s has too many rows (%lld) of %d channels", name, static_cast<long long>(a.rows), weight->channels));
    a.type = rows->precision;
    a.x = rowsOf(rows);   // (forward; the adjoint's rows are gradY)
    a.weight = matrixOf(weight);
    return a;
}
// what asks the device comes behind the checks
size_t onDevice(kernel::MxLinearArgs& a, bool adjoint)
{
    a.numSMs = Library::instance().smCount();
    a.status = Library::instance().statusWord();
    return adjoint ? kernel::mxLinearAdjointBytes(a) : kernel::mxLinearBytes(a);
}
void checkMxOffsets(const kernel::MxLinearArgs& a, const int32_t* offsets)
{
    if (offsets == nullptr && a.weight.matrices != 1) throw std::runtime_error("offsets is undefined");
}
const void* mxBias(const qmlp_tensor_t* bias, const kernel::MxLinearArgs& a, const char* name)
{
    kernel::ExpertArgs e{};
    e.experts = static_cast<int>(a.weight.matrices);
    e.channelsOut = static_cast<int>(a.weight.rows);
    e.type = a.type;
    return expertBias(bias, e, name);
}

} // namespace

extern "C" {

int qmlp_layer_norm_forward(const qmlp_tensor_t* input, const qmlp_tensor_t* weight, const qmlp_tensor_t* bias, float epsilon, qmlp_tensor_t* output, float* stats,
                            qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(input, "input", false);
    checkLike(output, input, "output", true);
    if (!(epsilon >= 0.f)) throw std::runtime_error("epsilon must not be negative");
    kernel::LayerNormArgs a = layerNorm(input);
    a.weight = vectorOf(weight, input, "weight");
    a.bias = vectorOf(bias, input, "bias");
    a.epsilon = epsilon;
    a.y = rowsOf(output);
    a.stats = stats;
    a.numSMs = Library::instance().smCount();
    a.status = Library::instance().statusWord();
    launch(KERNEL_ID_LAYER_NORM_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchLayerNormForward(a, s); });
    QMLP_CATCH
}
int qmlp_layer_norm_adjoint_memory(int64_t rows, int channels, int precision, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    if (rows < 0 || rows > MAX_ROWS || channels < 1 || channels > MAX_CHANNELS) throw std::runtime_error("layer norm of a matrix of an impossible size");
    *bytes = layerNormAdjointBytes(rows, channels, precision);
    QMLP_CATCH
}
int qmlp_layer_norm_adjoint(const qmlp_tensor_t* input, const qmlp_tensor_t* adj_output, const qmlp_tensor_t* weight, const float* stats, qmlp_tensor_t* adj_input,
                            qmlp_tensor_t* adj_weight, qmlp_tensor_t* adj_bias, qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    checkFeatures(input, "input", false);
    checkLike(adj_output, input, "adj_output", false);
    if (input->sizes[0] > 0) checkPointer(stats, "stats");
    kernel::LayerNormArgs a = layerNorm(input);
    a.weight = vectorOf(weight, input, "weight");
    a.gradY = rowsOf(adj_output);
    if (defined(adj_input)) {
        checkLike(adj_input, input, "adj_input", true);
        a.gradX = rowsOf(adj_input);
    }
    const kernel::Vector gw = vectorOf(adj_weight, input, "adj_weight"), gb = vectorOf(adj_bias, input, "adj_bias");
    a.gradWeight = const_cast<void*>(gw.data);
    a.gradWeightType = gw.type;
    a.gradBias = const_cast<void*>(gb.data);
    a.gradBiasType = gb.type;
    a.stats = const_cast<float*>(stats);
    if (a.gradWeight != nullptr || a.gradBias != nullptr) {
        checkScratch(tmp_memory, tmp_bytes, layerNormAdjointBytes(a.rows, a.channels, a.type));
        a.partial = static_cast<float*>(tmp_memory);
    }
    a.numSMs = Library::instance().smCount();
    a.status = Library::instance().statusWord();
    launch(KERNEL_ID_LAYER_NORM_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchLayerNormAdjoint(a, s); });
    QMLP_CATCH
}

int qmlp_embedding_forward(const qmlp_tensor_t* tokens, const qmlp_tensor_t* table, float scale, qmlp_tensor_t* output, qmlp_stream_t stream)
{
    QMLP_TRY
    checkTokens(tokens);
    checkFeatures(table, "table", false);
    checkFeatures(output, "output", true);
    checkDtype(output, table->precision, "output");
    checkSize(output, 0, tokens->sizes[0], "output");
    checkSize(output, 1, table->sizes[1], "output");
    kernel::EmbeddingArgs a{};
    a.tokens = tokens->sizes[0];
    a.rows = table->sizes[0];
    a.channels = static_cast<int>(table->sizes[1]);
    a.type = table->precision;
    a.tokenType = tokens->precision;
    a.token = tokens->data;
    a.tokenStride = tokens->strides[0];
    a.scale = scale;
    a.table = rowsOf(table);
    a.y = rowsOf(output);
    launch(KERNEL_ID_EMBEDDING_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchEmbeddingForward(a, s); });
    QMLP_CATCH
}
int qmlp_embedding_adjoint_memory(int64_t tokens, int64_t rows, int channels, int precision, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    if (tokens < 0 || tokens > MAX_SORTED || rows < 0 || rows > MAX_ROWS || channels < 1 || channels > MAX_CHANNELS)
        throw std::runtime_error("embedding of an impossible size");
    *bytes = kernel::embeddingAdjointBytes(tokens, rows, channels, precision, Library::instance().smCount());
    QMLP_CATCH
}
int qmlp_embedding_adjoint(const qmlp_tensor_t* tokens, const qmlp_tensor_t* adj_output, float scale, qmlp_tensor_t* adj_table, qmlp_stream_t stream, void* tmp_memory,
                           size_t tmp_bytes)
{
    QMLP_TRY
    checkTokens(tokens);
    if (tokens->sizes[0] > MAX_SORTED) throw std::runtime_error(format("tokens has too many entries (%lld)", static_cast<long long>(tokens->sizes[0])));
    checkFeatures(adj_table, "adj_table", true);
    checkFeatures(adj_output, "adj_output", false);
    checkDtype(adj_output, adj_table->precision, "adj_output");
    checkSize(adj_output, 0, tokens->sizes[0], "adj_output");
    checkSize(adj_output, 1, adj_table->sizes[1], "adj_output");
    kernel::EmbeddingArgs a{};
    a.tokens = tokens->sizes[0];
    a.rows = adj_table->sizes[0];
    a.channels = static_cast<int>(adj_table->sizes[1]);
    a.type = adj_table->precision;
    a.tokenType = tokens->precision;
    a.token = tokens->data;
    a.tokenStride = tokens->strides[0];
    a.scale = scale;
    a.gradY = rowsOf(adj_output);
    a.gradTable = rowsOf(adj_table);
    a.numSMs = Library::instance().smCount();
    checkScratch(tmp_memory, tmp_bytes, kernel::embeddingAdjointBytes(a.tokens, a.rows, a.channels, a.type, a.numSMs));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_EMBEDDING_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchEmbeddingAdjoint(a, s); });
    QMLP_CATCH
}

int qmlp_route_memory(const qmlp_routing_t* routing, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    checkRouting(routing);
    *bytes = kernel::routeBytes(routing->tokens, routing->num_experts, routing->chosen);
    QMLP_CATCH
}
static kernel::RouteArgs routeArgs(const qmlp_tensor_t* logits, int normalize, const qmlp_routing_t* r)
{
    checkRouting(r);
    checkFeatures(logits, "logits", false);
    checkSize(logits, 0, r->tokens, "logits");
    checkSize(logits, 1, r->num_experts, "logits");
    kernel::RouteArgs a{};
    a.tokens = r->tokens;
    a.experts = r->num_experts;
    a.chosen = r->chosen;
    a.type = logits->precision;
    a.normalize = normalize;
    a.logits = rowsOf(logits);
    a.weights = r->weights;
    a.expert = r->experts;
    a.order = r->order;
    a.position = r->positions;
    a.offsets = r->offsets;
    if (a.tokens > 0) {
        checkPointer(a.weights, "weights");
        checkPointer(a.expert, "experts");
    }
    return a;
}
int qmlp_route_forward(const qmlp_tensor_t* logits, int normalize, qmlp_routing_t* routing, qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    kernel::RouteArgs a = routeArgs(logits, normalize, routing);
    checkPointer(a.offsets, "offsets");
    if (a.tokens > 0) {
        checkPointer(a.order, "order");
        checkPointer(a.position, "positions");
    }
    checkScratch(tmp_memory, tmp_bytes, kernel::routeBytes(a.tokens, a.experts, a.chosen));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_ROUTE_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchRouteForward(a, s); });
    QMLP_CATCH
}
int qmlp_route_adjoint(const qmlp_tensor_t* logits, int normalize, const qmlp_routing_t* routing, const float* adj_weights, qmlp_tensor_t* adj_logits, qmlp_stream_t stream)
{
    QMLP_TRY
    kernel::RouteArgs a = routeArgs(logits, normalize, routing);
    checkLike(adj_logits, logits, "adj_logits", true);
    if (a.tokens > 0) checkPointer(adj_weights, "adj_weights");
    a.gradWeights = adj_weights;
    a.gradLogits = rowsOf(adj_logits);
    launch(KERNEL_ID_ROUTE_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchRouteAdjoint(a, s); });
    QMLP_CATCH
}

int qmlp_dispatch_forward(const qmlp_tensor_t* input, const qmlp_routing_t* routing, qmlp_tensor_t* rows, qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(input, "input", false);
    kernel::ExchangeArgs a = exchange(routing, input);
    checkSize(input, 0, a.tokens, "input");
    checkSlots(rows, routing, input, "rows", true);
    if (a.tokens > 0) checkPointer(a.order, "order");
    a.x = rowsOf(input);
    a.rows = rowsOf(rows);
    launch(KERNEL_ID_DISPATCH_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchDispatch(a, s); });
    QMLP_CATCH
}
int qmlp_dispatch_adjoint(const qmlp_tensor_t* adj_rows, const qmlp_routing_t* routing, qmlp_tensor_t* adj_input, qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(adj_input, "adj_input", true);
    kernel::ExchangeArgs a = exchange(routing, adj_input);
    checkSize(adj_input, 0, a.tokens, "adj_input");
    checkSlots(adj_rows, routing, adj_input, "adj_rows", false);
    if (a.tokens > 0) checkPointer(a.position, "positions");
    a.gradX = rowsOf(adj_input);
    a.gradRows = rowsOf(adj_rows);
    launch(KERNEL_ID_DISPATCH_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchDispatchAdjoint(a, s); });
    QMLP_CATCH
}
int qmlp_combine_forward(const qmlp_tensor_t* rows, const qmlp_routing_t* routing, qmlp_tensor_t* output, qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(output, "output", true);
    kernel::ExchangeArgs a = exchange(routing, output);
    checkSize(output, 0, a.tokens, "output");
    checkSlots(rows, routing, output, "rows", false);
    if (a.tokens > 0) {
        checkPointer(a.position, "positions");
        checkPointer(a.weights, "weights");
    }
    a.x = rowsOf(output);
    a.rows = rowsOf(rows);
    launch(KERNEL_ID_COMBINE_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchCombine(a, s); });
    QMLP_CATCH
}
int qmlp_combine_adjoint(const qmlp_tensor_t* rows, const qmlp_tensor_t* adj_output, const qmlp_routing_t* routing, qmlp_tensor_t* adj_rows, float* adj_weights,
                         qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(adj_output, "adj_output", false);
    kernel::ExchangeArgs a = exchange(routing, adj_output);
    checkSize(adj_output, 0, a.tokens, "adj_output");
    checkSlots(rows, routing, adj_output, "rows", false);
    if (a.tokens > 0) {
        checkPointer(a.position, "positions");
        checkPointer(a.weights, "weights");
    }
    a.gradX = rowsOf(adj_output);
    a.rows = rowsOf(rows);
    if (defined(adj_rows)) {
        checkSlots(adj_rows, routing, adj_output, "adj_rows", true);
        if (a.tokens > 0) checkPointer(a.order, "order");
        a.gradRows = rowsOf(adj_rows);
    }
    a.gradWeights = adj_weights;
    if (a.gradRows.data == nullptr && a.gradWeights == nullptr) return QMLP_OK;
    launch(KERNEL_ID_COMBINE_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchCombineAdjoint(a, s); });
    QMLP_CATCH
}

int qmlp_expert_linear_forward_memory(const qmlp_tensor_t* input, const qmlp_tensor_t* weight, int num_experts, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    kernel::ExpertArgs a = experts(input, weight, num_experts);
    a.numSMs = Library::instance().smCount();
    *bytes = kernel::expertBytes(a, false);
    QMLP_CATCH
}
int qmlp_expert_linear_forward(const qmlp_tensor_t* input, const qmlp_tensor_t* weight, const int32_t* offsets, int num_experts, const qmlp_tensor_t* bias,
                               qmlp_tensor_t* output, qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    kernel::ExpertArgs a = experts(input, weight, num_experts);
    checkPointer(offsets, "offsets");
    a.bias = expertBias(bias, a, "bias");
    checkFeatures(output, "output", true);
    checkDtype(output, a.type, "output");
    checkSize(output, 0, a.rows, "output");
    checkSize(output, 1, a.channelsOut, "output");
    a.offsets = offsets;
    a.y = rowsOf(output);
    a.numSMs = Library::instance().smCount();
    a.status = Library::instance().statusWord();
    checkScratch(tmp_memory, tmp_bytes, kernel::expertBytes(a, false));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_EXPERT_LINEAR_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchExpertForward(a, s); });
    QMLP_CATCH
}
int qmlp_expert_linear_adjoint_memory(const qmlp_tensor_t* input, const qmlp_tensor_t* adj_output, const qmlp_tensor_t* weight, int num_experts, int adjoint_flags,
                                      size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    kernel::ExpertArgs a = experts(input, weight, num_experts);
    expertGradients(a, adj_output, input);
    a.numSMs = Library::instance().smCount();
    char wanted = 0;   // (only whether a gradient is wanted enters the size)
    if (adjoint_flags & QMLP_GRADIENTS_INPUT) a.gradX.data = &wanted;
    if (adjoint_flags & QMLP_GRADIENTS_NETWORK_WEIGHTS) a.gradWeight = &wanted;
    *bytes = kernel::expertBytes(a, true);
    QMLP_CATCH
}
int qmlp_expert_linear_adjoint(const qmlp_tensor_t* input, const qmlp_tensor_t* adj_output, const qmlp_tensor_t* weight, const int32_t* offsets, int num_experts,
                               qmlp_tensor_t* adj_input, qmlp_tensor_t* adj_weight, qmlp_tensor_t* adj_bias, qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    kernel::ExpertArgs a = experts(input, weight, num_experts);
    checkPointer(offsets, "offsets");
    expertGradients(a, adj_output, input);
    a.offsets = offsets;
    if (defined(adj_input)) {
        checkLike(adj_input, input, "adj_input", true);
        a.gradX = rowsOf(adj_input);
    }
    if (defined(adj_weight)) {
        checkLike(adj_weight, weight, "adj_weight", true);
        if (adj_weight->sizes[0] > 1 && adj_weight->strides[0] != adj_weight->sizes[1]) throw std::runtime_error("adj_weight must be contiguous");
        a.gradWeight = adj_weight->data;
    }
    a.gradBias = const_cast<void*>(expertBias(adj_bias, a, "adj_bias"));
    a.numSMs = Library::instance().smCount();
    a.status = Library::instance().statusWord();
    checkScratch(tmp_memory, tmp_bytes, kernel::expertBytes(a, true));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_EXPERT_LINEAR_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchExpertAdjoint(a, s); });
    QMLP_CATCH
}

int qmlp_dropout(const qmlp_tensor_t* input, const qmlp_tensor_t* residual, double probability, uint64_t seed, uint64_t offset, const int64_t* step,
                 qmlp_tensor_t* output, qmlp_stream_t stream)
{
    QMLP_TRY
    checkFeatures(input, "input", false);
    checkLike(output, input, "output", true);
    if (!(probability >= 0. && probability <= 1.)) throw std::runtime_error("probability must be between 0 and 1");
    kernel::DropoutArgs a{};
    a.rows = input->sizes[0];
    a.channels = static_cast<int>(input->sizes[1]);
    a.type = input->precision;
    a.x = rowsOf(input);
    if (defined(residual)) {
        checkLike(residual, input, "residual", false);
        a.residual = rowsOf(residual);
    }
    a.y = rowsOf(output);
    a.cut = static_cast<unsigned>(std::nearbyint(probability * 65536.));
    a.seed = seed;
    a.offset = offset;
    a.step = reinterpret_cast<const long long*>(step);
    launch(KERNEL_ID_DROPOUT, stream, [&](cudaStream_t s) { return kernel::launchDropout(a, s); });
    QMLP_CATCH
}

int qmlp_mx_memory(int64_t matrices, int64_t rows, int channels, size_t* code_bytes, size_t* scale_bytes)
{
    QMLP_TRY
    checkPointer(code_bytes, "code_bytes");
    checkPointer(scale_bytes, "scale_bytes");
    alignas(16) uint8_t nothing[16];
    const qmlp_mx_t m{matrices, rows, channels, nothing, nothing};
    checkMx(&m, "matrix");
    *code_bytes = static_cast<size_t>(matrices * rows) * kernel::mxCodeBytes(channels);
    *scale_bytes = static_cast<size_t>(matrices) * kernel::mxTiles(rows) * kernel::mxTiles(channels) * kernel::MX_TILE_BYTES;
    QMLP_CATCH
}
int qmlp_mx_quantize(const qmlp_tensor_t* input, qmlp_mx_t* output, qmlp_stream_t stream)
{
    QMLP_TRY
    checkMx(output, "output");
    checkMxFeatures(input, output, "input", false);
    launch(KERNEL_ID_MX_QUANTIZE, stream, [&](cudaStream_t s) { return kernel::launchMxQuantize(matrixOf(output), input->precision, rowsOf(input), s); });
    QMLP_CATCH
}
int qmlp_mx_dequantize(const qmlp_mx_t* input, qmlp_tensor_t* output, qmlp_stream_t stream)
{
    QMLP_TRY
    checkMx(input, "input");
    checkMxFeatures(output, input, "output", true);
    launch(KERNEL_ID_MX_DEQUANTIZE, stream, [&](cudaStream_t s) { return kernel::launchMxDequantize(matrixOf(input), output->precision, rowsOf(output), s); });
    QMLP_CATCH
}

int qmlp_mx_linear_forward_memory(const qmlp_tensor_t* input, const qmlp_mx_t* weight, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    checkPointer(weight, "weight");
    kernel::MxLinearArgs a = mxLinear(input, weight, weight->channels, "input");
    *bytes = onDevice(a, false);
    QMLP_CATCH
}
int qmlp_mx_linear_forward(const qmlp_tensor_t* input, const qmlp_mx_t* weight, const int32_t* offsets, const qmlp_tensor_t* bias, qmlp_tensor_t* output,
                           qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    checkPointer(weight, "weight");
    kernel::MxLinearArgs a = mxLinear(input, weight, weight->channels, "input");
    checkMxOffsets(a, offsets);
    a.bias = mxBias(bias, a, "bias");
    checkFeatures(output, "output", true);
    checkDtype(output, a.type, "output");
    checkSize(output, 0, a.rows, "output");
    checkSize(output, 1, weight->rows, "output");
    a.offsets = offsets;
    a.y = rowsOf(output);
    checkScratch(tmp_memory, tmp_bytes, onDevice(a, false));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_MX_LINEAR_FORWARD, stream, [&](cudaStream_t s) { return kernel::launchMxLinear(a, s); });
    QMLP_CATCH
}
int qmlp_mx_linear_adjoint_memory(const qmlp_tensor_t* adj_output, const qmlp_mx_t* weight, int adjoint_flags, size_t* bytes)
{
    QMLP_TRY
    checkPointer(bytes, "bytes");
    checkPointer(weight, "weight");
    kernel::MxLinearArgs a = mxLinear(adj_output, weight, weight->rows, "adj_output");
    a.gradY = rowsOf(adj_output);
    char wanted = 0;   // (only whether a gradient is wanted enters the size)
    if (adjoint_flags & QMLP_GRADIENTS_INPUT) a.gradX.data = &wanted;
    *bytes = onDevice(a, true);
    QMLP_CATCH
}
int qmlp_mx_linear_adjoint(const qmlp_tensor_t* adj_output, const qmlp_mx_t* weight, const int32_t* offsets, qmlp_tensor_t* adj_input, qmlp_tensor_t* adj_bias,
                           qmlp_stream_t stream, void* tmp_memory, size_t tmp_bytes)
{
    QMLP_TRY
    checkPointer(weight, "weight");
    kernel::MxLinearArgs a = mxLinear(adj_output, weight, weight->rows, "adj_output");
    checkMxOffsets(a, offsets);
    a.offsets = offsets;
    a.gradY = rowsOf(adj_output);
    if (defined(adj_input)) {
        checkFeatures(adj_input, "adj_input", true);
        checkDtype(adj_input, a.type, "adj_input");
        checkSize(adj_input, 0, a.rows, "adj_input");
        checkSize(adj_input, 1, weight->channels, "adj_input");
        a.gradX = rowsOf(adj_input);
    }
    a.gradBias = const_cast<void*>(mxBias(adj_bias, a, "adj_bias"));
    checkScratch(tmp_memory, tmp_bytes, onDevice(a, true));
    a.scratch = tmp_memory;
    launch(KERNEL_ID_MX_LINEAR_ADJOINT, stream, [&](cudaStream_t s) { return kernel::launchMxLinearAdjoint(a, s); });
    QMLP_CATCH
}

} // extern "C"
