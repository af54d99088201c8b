// The operators on feature rows in PyTorch: torch.ops.qmlp_b200.{layer_norm, embedding, route, dispatch, combine, expert_linear}_forward
// and _adjoint, with their autograd nodes. Included by calls.cpp (whose helpers it uses); schemas in qmlp/ops.py.
//
// Every operator takes (..., channels) tensors; the leading dimensions are rows. A tensor whose rows the kernels cannot walk (elements of
// a row not side by side, leading dimensions that are no single stride) is copied first.
#pragma once

// ---- views -------------------------------------------------------------------------------------------------------------
int precisionOf(const Tensor& t)
{
    switch (t.scalar_type()) {
    case torch::kFloat32: return QMLP_FLOAT;
    case torch::kFloat16: return QMLP_HALF;
    case torch::kBFloat16: return QMLP_BFLOAT16;
    case torch::kInt32: return QMLP_INT32;
    case torch::kInt64: return QMLP_INT64;
    default: raiseError(std::string("unsupported dtype ") + c10::toString(t.scalar_type()));
    }
}
// (rows, channels) with the elements of a row side by side
Tensor asRows(const Tensor& t)
{
    if (t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= 0)) return t;
    if (t.dim() < 1) raiseError("a tensor of at least one dimension is needed");
    const int64_t channels = t.size(-1);
    const Tensor r = t.reshape({channels > 0 ? t.numel() / channels : 0, channels});
    return r.stride(1) == 1 || channels == 1 ? r : r.contiguous();
}
qmlp_tensor_t viewOf(const Tensor& t)
{
    qmlp_tensor_t v{};
    if (!t.defined()) return v;
    if (!t.is_cuda()) raiseError("tensor must live on a CUDA device");
    if (t.dim() < 1 || t.dim() > 2) raiseError("only 1-D and 2-D tensors are supported");
    v.precision = precisionOf(t);
    v.data = t.data_ptr();
    v.ndim = static_cast<int>(t.dim());
    for (int i = 0; i < v.ndim; ++i) {
        v.sizes[i] = t.size(i);
        v.strides[i] = t.stride(i);
    }
    return v;
}
// all on one CUDA device, which becomes the current one
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    template <class... T>
    explicit OnDevice(const Tensor& first, const T&... more)
    {
        if (!first.is_cuda()) raiseError("tensor must live on a CUDA device");
        (same(first, more), ...);
        if (first.device().index() != c10::cuda::current_device()) guard.set_index(first.device().index());
    }
    static void same(const Tensor& first, const Tensor& t)
    {
        if (t.defined() && t.device() != first.device()) raiseError("all tensors must live on one CUDA device");
    }
    static void same(const Tensor& first, const OptTensor& t)
    {
        if (t.has_value()) same(first, *t);
    }
};
// memory on the device of `like`, a CUDA tensor (below the dispatcher, which takes as long as the allocation itself)
Tensor emptyOn(at::IntArrayRef sizes, c10::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
Tensor emptyAs(at::IntArrayRef sizes, const Tensor& like) { return emptyOn(sizes, like.scalar_type(), like); }
struct ScratchMemory {
    Tensor memory;
    size_t bytes;
    ScratchMemory(size_t n, const Tensor& like) : bytes(n)
    {
        if (n > 0) memory = emptyOn({static_cast<int64_t>(n)}, torch::kUInt8, like);
    }
    void* data() const { return bytes > 0 ? memory.data_ptr() : nullptr; }
};
// a parameter of a layer, if there is one: its dimensions, the last of them `channels` (no dimension would read as no parameter)
void checkParameter(const OptTensor& t, int64_t dim, const c10::SymInt& channels, const char* name)
{
    if (!t.has_value() || !t->defined()) return;
    if (t->dim() != dim) raiseError(std::string(name) + " has the wrong dimension, expected " + std::to_string(dim) + " but got " + std::to_string(t->dim()));
    if (t->sym_size(-1) != channels) raiseError(std::string(name) + " has the wrong number of channels");
}
Tensor contiguousOf(const OptTensor& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }
Tensor emptyLike(const Tensor& t) { return emptyAs(t.sizes(), t); }
Tensor emptyFloat(at::IntArrayRef sizes, const Tensor& like) { return emptyOn(sizes, torch::kFloat32, like); }
Tensor emptyInt(at::IntArrayRef sizes, const Tensor& like) { return emptyOn(sizes, torch::kInt32, like); }
Tensor nothing(const Tensor& like) { return at::empty({0}, like.options()); }   // in the place of a gradient that is not asked for

// ---- layer norm ----------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> layerNormForward(const Tensor& input, const OptTensor& weight, const OptTensor& bias, double epsilon)
{
    const OnDevice on(input, weight, bias);
    const Tensor x = asRows(input);
    checkParameter(weight, 1, x.size(1), "weight");
    checkParameter(bias, 1, x.size(1), "bias");
    const Tensor w = contiguousOf(weight), b = contiguousOf(bias);
    Tensor y = emptyLike(input), stats = emptyFloat({2, x.size(0)}, x);
    const Tensor rows = y.dim() == 2 ? y : y.view(x.sizes());
    const qmlp_tensor_t vx = viewOf(x), vw = viewOf(w), vb = viewOf(b);
    qmlp_tensor_t vy = viewOf(rows);
    check(api.layer_norm_forward(&vx, &vw, &vb, static_cast<float>(epsilon), &vy, static_cast<float*>(stats.data_ptr()), currentStream()));
    return {y, stats};
}
// what the forward pass left: means and reciprocal deviations of the rows
void checkStats(const Tensor& stats, const c10::SymInt& rows)
{
    if (stats.scalar_type() != torch::kFloat32 || stats.dim() != 2 || stats.sym_size(0) != 2 || stats.sym_size(1) != rows || !stats.is_contiguous())
        raiseError("stats must be a contiguous float32 tensor (2, rows)");
}
std::tuple<Tensor, Tensor, Tensor> layerNormAdjoint(const Tensor& input, const Tensor& adjOutput, const OptTensor& weight, const OptTensor& bias, const Tensor& stats,
                                                    bool wantInput, bool wantWeight, bool wantBias)
{
    const OnDevice on(input, adjOutput, weight, bias, stats);
    const Tensor x = asRows(input), g = asRows(adjOutput), w = contiguousOf(weight);
    checkParameter(weight, 1, x.size(1), "weight");
    checkParameter(bias, 1, x.size(1), "bias");
    checkStats(stats, x.size(0));
    const bool haveWeight = wantWeight && w.defined(), haveBias = wantBias && bias.has_value() && bias->defined();
    Tensor dx = wantInput ? emptyLike(input) : Tensor(), dw = haveWeight ? emptyLike(w) : Tensor(), db = haveBias ? emptyLike(*bias) : Tensor();
    size_t bytes = 0;
    if (haveWeight || haveBias) check(api.layer_norm_adjoint_memory(x.size(0), static_cast<int>(x.size(1)), precisionOf(x), &bytes));
    const ScratchMemory tmp(bytes, x);
    const qmlp_tensor_t vx = viewOf(x), vg = viewOf(g), vw = viewOf(w);
    qmlp_tensor_t vdx = viewOf(wantInput ? dx.view(x.sizes()) : dx), vdw = viewOf(dw), vdb = viewOf(db);
    check(api.layer_norm_adjoint(&vx, &vg, &vw, static_cast<const float*>(stats.data_ptr()), &vdx, &vdw, &vdb, currentStream(), tmp.data(), bytes));
    return {wantInput ? dx : nothing(input), haveWeight ? dw : nothing(input), haveBias ? db : nothing(input)};
}

// ---- embedding -----------------------------------------------------------------------------------------------------------
std::vector<int64_t> rowShape(const Tensor& tokens, int64_t channels)
{
    std::vector<int64_t> shape = tokens.sizes().vec();
    shape.push_back(channels);
    return shape;
}
Tensor flatTokens(const Tensor& tokens) { return tokens.dim() == 1 ? tokens : tokens.reshape({-1}); }
Tensor embeddingForward(const Tensor& tokens, const Tensor& table, double scale)
{
    const OnDevice on(table, tokens);
    if (table.dim() != 2) raiseError("table must be a matrix of rows and channels");
    const Tensor t = flatTokens(tokens), rows = asRows(table);
    Tensor y = emptyAs(rowShape(tokens, table.size(1)), table);
    const qmlp_tensor_t vt = viewOf(t), vr = viewOf(rows);
    qmlp_tensor_t vy = viewOf(y.dim() == 2 ? y : y.view({t.size(0), table.size(1)}));
    check(api.embedding_forward(&vt, &vr, static_cast<float>(scale), &vy, currentStream()));
    return y;
}
Tensor embeddingAdjoint(const Tensor& tokens, const Tensor& adjOutput, int64_t rows, double scale)
{
    const OnDevice on(adjOutput, tokens);
    const Tensor t = flatTokens(tokens), g = asRows(adjOutput);
    Tensor table = emptyAs({rows, g.size(1)}, g);
    size_t bytes = 0;
    check(api.embedding_adjoint_memory(t.size(0), rows, static_cast<int>(g.size(1)), precisionOf(g), &bytes));
    const ScratchMemory tmp(bytes, g);
    const qmlp_tensor_t vt = viewOf(t), vg = viewOf(g);
    qmlp_tensor_t vr = viewOf(table);
    check(api.embedding_adjoint(&vt, &vg, static_cast<float>(scale), &vr, currentStream(), tmp.data(), bytes));
    return table;
}

// ---- routing ---------------------------------------------------------------------------------------------------------------
int* intData(const Tensor& t, const char* name)
{
    if (t.scalar_type() != torch::kInt32 || !t.is_contiguous()) raiseError(std::string(name) + " must be a contiguous int32 tensor");
    return static_cast<int*>(t.data_ptr());
}
float* floatData(const Tensor& t, const char* name)
{
    if (t.scalar_type() != torch::kFloat32 || !t.is_contiguous()) raiseError(std::string(name) + " must be a contiguous float32 tensor");
    return static_cast<float*>(t.data_ptr());
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> routeForward(const Tensor& logits, int64_t chosen, bool normalize)
{
    const OnDevice on(logits);
    if (logits.dim() != 2) raiseError("logits must be a matrix of rows and experts");
    const Tensor z = asRows(logits);
    const int64_t n = z.size(0), e = z.size(1);
    if (chosen < 1 || chosen > 32 || chosen > e || e > 1024) raiseError("a row chooses 1 to 32 of its experts, of which there are at most 1024");
    // (the schema promises results that share nothing: views of one allocation would do away with three of five)
    Tensor weights = emptyFloat({n, chosen}, z), experts = emptyInt({n, chosen}, z), positions = emptyInt({n, chosen}, z), order = emptyInt({n * chosen}, z),
           offsets = emptyInt({e + 1}, z);
    qmlp_routing_t r{n, static_cast<int32_t>(e), static_cast<int32_t>(chosen), static_cast<float*>(weights.data_ptr()), static_cast<int*>(experts.data_ptr()),
                     static_cast<int*>(order.data_ptr()), static_cast<int*>(positions.data_ptr()), static_cast<int*>(offsets.data_ptr())};
    size_t bytes = 0;
    check(api.route_memory(&r, &bytes));
    const ScratchMemory tmp(bytes, z);
    const qmlp_tensor_t vz = viewOf(z);
    check(api.route_forward(&vz, normalize, &r, currentStream(), tmp.data(), bytes));
    return {weights, experts, order, positions, offsets};
}
Tensor routeAdjoint(const Tensor& logits, bool normalize, const Tensor& weights, const Tensor& experts, const Tensor& adjWeights)
{
    const OnDevice on(logits, weights, experts, adjWeights);
    const Tensor z = asRows(logits), g = adjWeights.contiguous();
    if (weights.dim() != 2 || weights.size(0) != z.size(0) || !experts.sizes().equals(weights.sizes()) || !g.sizes().equals(weights.sizes()))
        raiseError("weights, experts and adj_weights must be (rows, chosen)");
    Tensor dz = emptyLike(z);
    qmlp_routing_t r{z.size(0), static_cast<int32_t>(z.size(1)), static_cast<int32_t>(weights.size(1)), floatData(weights, "weights"), intData(experts, "experts"),
                     nullptr, nullptr, nullptr};
    const qmlp_tensor_t vz = viewOf(z);
    qmlp_tensor_t vd = viewOf(dz);
    check(api.route_adjoint(&vz, normalize, &r, floatData(g, "adj_weights"), &vd, currentStream()));
    return dz;
}

// the arrays of a routing that the movement of rows needs
qmlp_routing_t routingOf(const Tensor& order, const Tensor& positions, const OptTensor& weights)
{
    if (positions.dim() != 2 || (order.defined() && (order.dim() != 1 || order.size(0) != positions.numel())))
        raiseError("order must have the entries of positions, which is (rows, chosen)");
    qmlp_routing_t r{};
    r.tokens = positions.size(0);
    r.chosen = static_cast<int32_t>(positions.size(1));
    r.num_experts = std::max<int32_t>(r.chosen, 1);   // (the number of experts does not matter here)
    r.positions = intData(positions, "positions");
    if (order.defined()) r.order = intData(order, "order");
    if (weights.has_value()) {
        if (!weights->sizes().equals(positions.sizes())) raiseError("weights must be (rows, chosen)");
        r.weights = floatData(*weights, "weights");
    }
    return r;
}
Tensor dispatchForward(const Tensor& input, const Tensor& order, const Tensor& positions)
{
    const OnDevice on(input, order, positions);
    const Tensor x = asRows(input);
    const qmlp_routing_t r = routingOf(order, positions, std::nullopt);
    Tensor rows = emptyAs({order.size(0), x.size(1)}, x);
    const qmlp_tensor_t vx = viewOf(x);
    qmlp_tensor_t vr = viewOf(rows);
    check(api.dispatch_forward(&vx, &r, &vr, currentStream()));
    return rows;
}
Tensor dispatchAdjoint(const Tensor& adjRows, const Tensor& positions)
{
    const OnDevice on(adjRows, positions);
    const Tensor g = asRows(adjRows);
    const qmlp_routing_t r = routingOf(Tensor(), positions, std::nullopt);
    Tensor dx = emptyAs({positions.size(0), g.size(1)}, g);
    const qmlp_tensor_t vg = viewOf(g);
    qmlp_tensor_t vd = viewOf(dx);
    check(api.dispatch_adjoint(&vg, &r, &vd, currentStream()));
    return dx;
}
// (the order of the slots is an argument for the sake of the gradient)
Tensor combineForward(const Tensor& rows, const Tensor& weights, const Tensor& order, const Tensor& positions)
{
    const OnDevice on(rows, weights, order, positions);
    const Tensor y = asRows(rows);
    const Tensor w = weights.contiguous();
    const qmlp_routing_t r = routingOf(order, positions, w);
    Tensor out = emptyAs({positions.size(0), y.size(1)}, y);
    const qmlp_tensor_t vy = viewOf(y);
    qmlp_tensor_t vo = viewOf(out);
    check(api.combine_forward(&vy, &r, &vo, currentStream()));
    return out;
}
std::tuple<Tensor, Tensor> combineAdjoint(const Tensor& rows, const Tensor& adjOutput, const Tensor& weights, const Tensor& order, const Tensor& positions, bool wantRows,
                                          bool wantWeights)
{
    const OnDevice on(rows, adjOutput, weights, order, positions);
    const Tensor y = asRows(rows), g = asRows(adjOutput), w = weights.contiguous();
    const qmlp_routing_t r = routingOf(order, positions, w);
    Tensor dy = wantRows ? emptyLike(y) : Tensor(), dw = wantWeights ? emptyFloat(w.sizes(), w) : Tensor();
    const qmlp_tensor_t vy = viewOf(y), vg = viewOf(g);
    qmlp_tensor_t vd = viewOf(dy);
    check(api.combine_adjoint(&vy, &vg, &r, &vd, wantWeights ? static_cast<float*>(dw.data_ptr()) : nullptr, currentStream()));
    return {wantRows ? dy.view(rows.sizes()) : nothing(rows), wantWeights ? dw : nothing(weights)};
}

// ---- products grouped by expert ----------------------------------------------------------------------------------------------
// (experts, channels out, channels in) -> the rows of all matrices, one below the other
Tensor matricesOf(const Tensor& weight)
{
    if (weight.dim() != 3) raiseError("weight must be (experts, channels out, channels in)");
    return weight.contiguous().view({weight.size(0) * weight.size(1), weight.size(2)});
}
int* offsetsOf(const Tensor& offsets, const Tensor& weight)
{
    if (offsets.dim() != 1 || offsets.size(0) != weight.size(0) + 1) raiseError("offsets must have one entry per expert and one more");
    return intData(offsets, "offsets");
}
Tensor expertLinearForward(const Tensor& input, const Tensor& weight, const Tensor& offsets, const OptTensor& bias)
{
    const OnDevice on(input, weight, offsets, bias);
    const Tensor x = asRows(input), w = matricesOf(weight);
    checkParameter(bias, 2, weight.size(1), "bias");
    const Tensor b = contiguousOf(bias);
    const int experts = static_cast<int>(weight.size(0));
    Tensor y = emptyAs({x.size(0), weight.size(1)}, x);
    const qmlp_tensor_t vx = viewOf(x), vw = viewOf(w), vb = viewOf(b);
    qmlp_tensor_t vy = viewOf(y);
    size_t bytes = 0;
    check(api.expert_linear_forward_memory(&vx, &vw, experts, &bytes));
    const ScratchMemory tmp(bytes, x);
    check(api.expert_linear_forward(&vx, &vw, offsetsOf(offsets, weight), experts, &vb, &vy, currentStream(), tmp.data(), bytes));
    return y;
}
std::tuple<Tensor, Tensor, Tensor> expertLinearAdjoint(const Tensor& input, const Tensor& adjOutput, const Tensor& weight, const Tensor& offsets, bool wantInput,
                                                       bool wantWeight, bool wantBias)
{
    const OnDevice on(input, adjOutput, weight, offsets);
    const Tensor x = asRows(input), g = asRows(adjOutput), w = matricesOf(weight);
    const int experts = static_cast<int>(weight.size(0));
    Tensor dx = wantInput ? emptyLike(x) : Tensor(), dw = wantWeight ? emptyAs(weight.sizes(), w) : Tensor();
    Tensor db = wantBias ? emptyAs({weight.size(0), weight.size(1)}, w) : Tensor();
    const qmlp_tensor_t vx = viewOf(x), vg = viewOf(g), vw = viewOf(w);
    qmlp_tensor_t vdx = viewOf(dx), vdw = viewOf(wantWeight ? dw.view(w.sizes()) : dw), vdb = viewOf(db);
    size_t bytes = 0;
    check(api.expert_linear_adjoint_memory(&vx, &vg, &vw, experts, (wantInput ? QMLP_GRADIENTS_INPUT : 0) | (wantWeight ? QMLP_GRADIENTS_NETWORK_WEIGHTS : 0), &bytes));
    const ScratchMemory tmp(bytes, x);
    check(api.expert_linear_adjoint(&vx, &vg, &vw, offsetsOf(offsets, weight), experts, &vdx, &vdw, &vdb, currentStream(), tmp.data(), bytes));
    return {wantInput ? dx : nothing(input), wantWeight ? dw : nothing(weight), wantBias ? db : nothing(weight)};
}

// ---- autograd --------------------------------------------------------------------------------------------------------------
template <class F>
auto operatorHandle(const char* name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow((std::string("qmlp_b200::") + name).c_str(), "").typed<F>();
}
#define QMLP_CALL(name, function) ([]() -> const auto& { static const auto op = operatorHandle<decltype(function)>(name); return op; }())

// results of an adjoint operator, with a node that refuses a second differentiation
struct OnceFunction : torch::autograd::Function<OnceFunction> {
    static variable_list forward(AutogradContext* ctx, const std::string& op, const variable_list& results, at::TensorList)
    {
        ctx->saved_data["op"] = op;
        return results;
    }
    static variable_list backward(AutogradContext* ctx, variable_list) { raiseNotTwice(ctx->saved_data["op"].toStringRef().c_str()); }
};
variable_list once(const char* op, variable_list results, std::vector<Tensor> sources)
{
    std::vector<Tensor> wanted;
    for (auto& s : sources)
        if (differentiable(s)) wanted.push_back(s);
    if (!torch::GradMode::is_enabled() || wanted.empty()) return results;
    return OnceFunction::apply(std::string(op), results, at::TensorList(wanted));
}
// The operators have no forward-mode formula. A dual tensor, which torch.func.jvp makes too, is refused: below autograd its tangent would be lost.
bool hasTangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool hasTangent(const OptTensor& t) { return t.has_value() && hasTangent(*t); }
template <class... T>
void refuseTangents(const char* op, const T&... tensors)
{
    if ((hasTangent(tensors) || ...)) raiseError(std::string("qmlp_b200::") + op + " has no forward-mode derivative");
}
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& input, const OptTensor& weight, const OptTensor& bias, double epsilon)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        auto r = QMLP_CALL("layer_norm_forward", layerNormForward).call(input, weight, bias, epsilon);
        ctx->save_for_backward({input, weight.value_or(Tensor()), bias.value_or(Tensor()), std::get<1>(r)});
        ctx->mark_non_differentiable({std::get<1>(r)});
        ctx->set_materialize_grads(false);   // (a fill kernel for every output nobody differentiates)
        return {std::get<0>(r), std::get<1>(r)};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        if (!grad[0].defined()) return variable_list(4);
        const auto s = ctx->get_saved_variables();
        const bool wx = ctx->needs_input_grad(0), ww = s[1].defined() && ctx->needs_input_grad(1), wb = s[2].defined() && ctx->needs_input_grad(s[1].defined() ? 2 : 1);
        auto g = QMLP_CALL("layer_norm_adjoint", layerNormAdjoint).call(s[0], grad[0], optional(s[1]), optional(s[2]), s[3], wx, ww, wb);
        return {wx ? std::get<0>(g) : Tensor(), ww ? std::get<1>(g) : Tensor(), wb ? std::get<2>(g) : Tensor(), Tensor()};
    }
};
std::tuple<Tensor, Tensor> layerNormForwardAutograd(const Tensor& input, const OptTensor& weight, const OptTensor& bias, double epsilon)
{
    refuseTangents("layer_norm_forward", input, weight, bias);
    if (wantsNode(input, weight, bias)) {
        auto r = LayerNormFunction::apply(input, weight, bias, epsilon);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("layer_norm_forward", layerNormForward).call(input, weight, bias, epsilon);
}
std::tuple<Tensor, Tensor, Tensor> layerNormAdjointAutograd(const Tensor& input, const Tensor& adjOutput, const OptTensor& weight, const OptTensor& bias,
                                                            const Tensor& stats, bool wantInput, bool wantWeight, bool wantBias)
{
    refuseTangents("layer_norm_adjoint", input, adjOutput, weight, bias);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        auto g = QMLP_CALL("layer_norm_adjoint", layerNormAdjoint).call(input, adjOutput, weight, bias, stats, wantInput, wantWeight, wantBias);
        r = {std::get<0>(g), std::get<1>(g), std::get<2>(g)};
    }
    r = once("layer_norm_adjoint", r, {input, adjOutput, weight.value_or(Tensor()), bias.value_or(Tensor())});
    return {r[0], r[1], r[2]};
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& table, double scale)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({tokens});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        return QMLP_CALL("embedding_forward", embeddingForward).call(tokens, table, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        return {Tensor(), QMLP_CALL("embedding_adjoint", embeddingAdjoint).call(ctx->get_saved_variables()[0], grad[0], ctx->saved_data["rows"].toInt(),
                                                                                ctx->saved_data["scale"].toDouble()), Tensor()};
    }
};
Tensor embeddingForwardAutograd(const Tensor& tokens, const Tensor& table, double scale)
{
    refuseTangents("embedding_forward", table);
    if (wantsNode(table)) return EmbeddingFunction::apply(tokens, table, scale);
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("embedding_forward", embeddingForward).call(tokens, table, scale);
}
Tensor embeddingAdjointAutograd(const Tensor& tokens, const Tensor& adjOutput, int64_t rows, double scale)
{
    refuseTangents("embedding_adjoint", adjOutput);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = {QMLP_CALL("embedding_adjoint", embeddingAdjoint).call(tokens, adjOutput, rows, scale)};
    }
    return once("embedding_adjoint", r, {adjOutput})[0];
}

using RouteResult = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;
struct RouteFunction : torch::autograd::Function<RouteFunction> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t chosen, bool normalize)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [weights, experts, order, positions, offsets] = QMLP_CALL("route_forward", routeForward).call(logits, chosen, normalize);
        ctx->save_for_backward({logits, weights, experts});
        ctx->saved_data["normalize"] = normalize;
        ctx->mark_non_differentiable({experts, order, positions, offsets});
        ctx->set_materialize_grads(false);
        return {weights, experts, order, positions, offsets};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        if (!grad[0].defined()) return variable_list(3);
        const auto s = ctx->get_saved_variables();
        return {QMLP_CALL("route_adjoint", routeAdjoint).call(s[0], ctx->saved_data["normalize"].toBool(), s[1], s[2], grad[0]), Tensor(), Tensor()};
    }
};
RouteResult routeForwardAutograd(const Tensor& logits, int64_t chosen, bool normalize)
{
    refuseTangents("route_forward", logits);
    if (wantsNode(logits)) {
        auto r = RouteFunction::apply(logits, chosen, normalize);
        return {r[0], r[1], r[2], r[3], r[4]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("route_forward", routeForward).call(logits, chosen, normalize);
}
Tensor routeAdjointAutograd(const Tensor& logits, bool normalize, const Tensor& weights, const Tensor& experts, const Tensor& adjWeights)
{
    refuseTangents("route_adjoint", logits, weights, adjWeights);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = {QMLP_CALL("route_adjoint", routeAdjoint).call(logits, normalize, weights, experts, adjWeights)};
    }
    return once("route_adjoint", r, {logits, weights, adjWeights})[0];
}

struct DispatchFunction : torch::autograd::Function<DispatchFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& input, const Tensor& order, const Tensor& positions)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({positions});
        ctx->saved_data["shape"] = input.sizes().vec();
        return QMLP_CALL("dispatch_forward", dispatchForward).call(input, order, positions);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        const Tensor dx = QMLP_CALL("dispatch_adjoint", dispatchAdjoint).call(grad[0], ctx->get_saved_variables()[0]);
        return {dx.view(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor()};
    }
};
Tensor dispatchForwardAutograd(const Tensor& input, const Tensor& order, const Tensor& positions)
{
    refuseTangents("dispatch_forward", input);
    if (wantsNode(input)) return DispatchFunction::apply(input, order, positions);
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("dispatch_forward", dispatchForward).call(input, order, positions);
}
Tensor dispatchAdjointAutograd(const Tensor& adjRows, const Tensor& positions)
{
    refuseTangents("dispatch_adjoint", adjRows);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        r = {QMLP_CALL("dispatch_adjoint", dispatchAdjoint).call(adjRows, positions)};
    }
    return once("dispatch_adjoint", r, {adjRows})[0];
}

struct CombineFunction : torch::autograd::Function<CombineFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights, const Tensor& order, const Tensor& positions)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({rows, weights, order, positions});
        return QMLP_CALL("combine_forward", combineForward).call(rows, weights, order, positions);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        const auto s = ctx->get_saved_variables();
        const bool wr = ctx->needs_input_grad(0), ww = ctx->needs_input_grad(1);
        auto g = QMLP_CALL("combine_adjoint", combineAdjoint).call(s[0], grad[0], s[1], s[2], s[3], wr, ww);
        return {wr ? std::get<0>(g) : Tensor(), ww ? std::get<1>(g) : Tensor(), Tensor(), Tensor()};
    }
};
Tensor combineForwardAutograd(const Tensor& rows, const Tensor& weights, const Tensor& order, const Tensor& positions)
{
    refuseTangents("combine_forward", rows, weights);
    if (wantsNode(rows, weights)) return CombineFunction::apply(rows, weights, order, positions);
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("combine_forward", combineForward).call(rows, weights, order, positions);
}
std::tuple<Tensor, Tensor> combineAdjointAutograd(const Tensor& rows, const Tensor& adjOutput, const Tensor& weights, const Tensor& order, const Tensor& positions,
                                                  bool wantRows, bool wantWeights)
{
    refuseTangents("combine_adjoint", rows, adjOutput, weights);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        auto g = QMLP_CALL("combine_adjoint", combineAdjoint).call(rows, adjOutput, weights, order, positions, wantRows, wantWeights);
        r = {std::get<0>(g), std::get<1>(g)};
    }
    r = once("combine_adjoint", r, {rows, adjOutput, weights});
    return {r[0], r[1]};
}

struct ExpertLinearFunction : torch::autograd::Function<ExpertLinearFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& input, const Tensor& weight, const Tensor& offsets, const OptTensor& bias)
    {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({input, weight, offsets});
        ctx->saved_data["bias"] = bias.has_value() && bias->defined();
        return QMLP_CALL("expert_linear_forward", expertLinearForward).call(input, weight, offsets, bias);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grad)
    {
        const auto s = ctx->get_saved_variables();
        const bool wx = ctx->needs_input_grad(0), ww = ctx->needs_input_grad(1), wb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
        auto g = QMLP_CALL("expert_linear_adjoint", expertLinearAdjoint).call(s[0], grad[0], s[1], s[2], wx, ww, wb);
        return {wx ? std::get<0>(g).view(s[0].sizes()) : Tensor(), ww ? std::get<1>(g) : Tensor(), Tensor(), wb ? std::get<2>(g) : Tensor()};
    }
};
Tensor expertLinearForwardAutograd(const Tensor& input, const Tensor& weight, const Tensor& offsets, const OptTensor& bias)
{
    refuseTangents("expert_linear_forward", input, weight, bias);
    if (wantsNode(input, weight, bias)) return ExpertLinearFunction::apply(input, weight, offsets, bias);
    at::AutoDispatchBelowADInplaceOrView below;
    return QMLP_CALL("expert_linear_forward", expertLinearForward).call(input, weight, offsets, bias);
}
std::tuple<Tensor, Tensor, Tensor> expertLinearAdjointAutograd(const Tensor& input, const Tensor& adjOutput, const Tensor& weight, const Tensor& offsets, bool wantInput,
                                                               bool wantWeight, bool wantBias)
{
    refuseTangents("expert_linear_adjoint", input, adjOutput, weight);
    variable_list r;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        auto g = QMLP_CALL("expert_linear_adjoint", expertLinearAdjoint).call(input, adjOutput, weight, offsets, wantInput, wantWeight, wantBias);
        r = {std::get<0>(g), std::get<1>(g), std::get<2>(g)};
    }
    r = once("expert_linear_adjoint", r, {input, adjOutput, weight});
    return {r[0], r[1], r[2]};
}

// ---- shapes (meta tensors) ---------------------------------------------------------------------------------------------------
Tensor emptyOf(const Tensor& like, c10::SymIntArrayRef sizes) { return at::empty_symint(sizes, like.options().memory_format(c10::MemoryFormat::Contiguous)); }
Tensor emptyOf(const Tensor& like, c10::SymIntArrayRef sizes, c10::ScalarType type) { return at::empty_symint(sizes, like.options().dtype(type)); }
c10::SymInt rowsIn(const Tensor& t)
{
    if (t.dim() < 1) raiseError("a tensor of at least one dimension is needed");
    if (t.sym_size(-1) == 0) raiseError("a tensor of at least one channel is needed");   // (a division by zero ends the process)
    return t.sym_numel() / t.sym_size(-1);
}

std::tuple<Tensor, Tensor> layerNormForwardMeta(const Tensor& input, const OptTensor& weight, const OptTensor& bias, double)
{
    const c10::SymInt rows = rowsIn(input);
    checkParameter(weight, 1, input.sym_size(-1), "weight");
    checkParameter(bias, 1, input.sym_size(-1), "bias");
    return {emptyOf(input, input.sym_sizes()), emptyOf(input, {2, rows}, torch::kFloat32)};
}
std::tuple<Tensor, Tensor, Tensor> layerNormAdjointMeta(const Tensor& input, const Tensor&, const OptTensor& weight, const OptTensor& bias, const Tensor& stats, bool wantInput,
                                                        bool wantWeight, bool wantBias)
{
    const c10::SymInt rows = rowsIn(input);
    checkParameter(weight, 1, input.sym_size(-1), "weight");
    checkParameter(bias, 1, input.sym_size(-1), "bias");
    checkStats(stats, rows);
    return {wantInput ? emptyOf(input, input.sym_sizes()) : nothing(input), wantWeight && weight.has_value() ? at::empty_like(*weight) : nothing(input),
            wantBias && bias.has_value() ? at::empty_like(*bias) : nothing(input)};
}
Tensor embeddingForwardMeta(const Tensor& tokens, const Tensor& table, double)
{
    c10::SymDimVector shape(tokens.sym_sizes().begin(), tokens.sym_sizes().end());
    shape.push_back(table.sym_size(1));
    return emptyOf(table, shape);
}
Tensor embeddingAdjointMeta(const Tensor&, const Tensor& adjOutput, int64_t rows, double) { return emptyOf(adjOutput, {c10::SymInt(rows), adjOutput.sym_size(-1)}); }
RouteResult routeForwardMeta(const Tensor& logits, int64_t chosen, bool)
{
    const c10::SymInt n = logits.sym_size(0), e = logits.sym_size(1);
    return {emptyOf(logits, {n, c10::SymInt(chosen)}, torch::kFloat32), emptyOf(logits, {n, c10::SymInt(chosen)}, torch::kInt32), emptyOf(logits, {n * chosen}, torch::kInt32),
            emptyOf(logits, {n, c10::SymInt(chosen)}, torch::kInt32), emptyOf(logits, {e + 1}, torch::kInt32)};
}
Tensor routeAdjointMeta(const Tensor& logits, bool, const Tensor&, const Tensor&, const Tensor&) { return emptyOf(logits, logits.sym_sizes()); }
Tensor dispatchForwardMeta(const Tensor& input, const Tensor& order, const Tensor&) { return emptyOf(input, {order.sym_size(0), input.sym_size(-1)}); }
Tensor dispatchAdjointMeta(const Tensor& adjRows, const Tensor& positions) { return emptyOf(adjRows, {positions.sym_size(0), adjRows.sym_size(-1)}); }
Tensor combineForwardMeta(const Tensor& rows, const Tensor&, const Tensor&, const Tensor& positions) { return emptyOf(rows, {positions.sym_size(0), rows.sym_size(-1)}); }
std::tuple<Tensor, Tensor> combineAdjointMeta(const Tensor& rows, const Tensor&, const Tensor& weights, const Tensor&, const Tensor&, bool wantRows, bool wantWeights)
{
    return {wantRows ? emptyOf(rows, rows.sym_sizes()) : nothing(rows), wantWeights ? emptyOf(weights, weights.sym_sizes()) : nothing(weights)};
}
Tensor expertLinearForwardMeta(const Tensor& input, const Tensor& weight, const Tensor&, const OptTensor& bias)
{
    if (weight.dim() != 3) raiseError("weight must be (experts, channels out, channels in)");
    checkParameter(bias, 2, weight.sym_size(1), "bias");
    return emptyOf(input, {rowsIn(input), weight.sym_size(1)});
}
std::tuple<Tensor, Tensor, Tensor> expertLinearAdjointMeta(const Tensor& input, const Tensor&, const Tensor& weight, const Tensor&, bool wantInput, bool wantWeight,
                                                           bool wantBias)
{
    return {wantInput ? emptyOf(input, {rowsIn(input), input.sym_size(-1)}) : nothing(input), wantWeight ? emptyOf(weight, weight.sym_sizes()) : nothing(weight),
            wantBias ? emptyOf(weight, {weight.sym_size(0), weight.sym_size(1)}) : nothing(weight)};
}

#define QMLP_ROW_OPERATORS(X, suffix)                                                                                          \
    X("layer_norm_forward", layerNormForward##suffix) X("layer_norm_adjoint", layerNormAdjoint##suffix)                         \
    X("embedding_forward", embeddingForward##suffix) X("embedding_adjoint", embeddingAdjoint##suffix)                           \
    X("route_forward", routeForward##suffix) X("route_adjoint", routeAdjoint##suffix)                                           \
    X("dispatch_forward", dispatchForward##suffix) X("dispatch_adjoint", dispatchAdjoint##suffix)                               \
    X("combine_forward", combineForward##suffix) X("combine_adjoint", combineAdjoint##suffix)                                   \
    X("expert_linear_forward", expertLinearForward##suffix) X("expert_linear_adjoint", expertLinearAdjoint##suffix)
#define QMLP_IMPL(name, function) m->impl(name, function);

void registerRowOperators(c10::DispatchKey key)
{
    auto* m = new torch::Library(torch::Library::IMPL, "qmlp_b200", key, __FILE__, __LINE__);   // (lives as long as the process)
    if (key == c10::DispatchKey::CUDA) { QMLP_ROW_OPERATORS(QMLP_IMPL, ) }
    else if (key == c10::DispatchKey::Meta) { QMLP_ROW_OPERATORS(QMLP_IMPL, Meta) }
    else { QMLP_ROW_OPERATORS(QMLP_IMPL, Autograd) }
}

// ---- what qmlp/rows.py calls: the operators through the dispatcher, without the interpreter's detour -----------------------------
Tensor layerNorm(const Tensor& input, const OptTensor& weight, const OptTensor& bias, double epsilon)
{
    return std::get<0>(QMLP_CALL("layer_norm_forward", layerNormForward).call(input, weight, bias, epsilon));
}
Tensor embedding(const Tensor& tokens, const Tensor& table, double scale) { return QMLP_CALL("embedding_forward", embeddingForward).call(tokens, table, scale); }
RouteResult route(const Tensor& logits, int64_t chosen, bool normalize) { return QMLP_CALL("route_forward", routeForward).call(logits, chosen, normalize); }
Tensor dispatchRows(const Tensor& input, const Tensor& order, const Tensor& positions)
{
    return QMLP_CALL("dispatch_forward", dispatchForward).call(input, order, positions);
}
Tensor combineRows(const Tensor& rows, const Tensor& weights, const Tensor& order, const Tensor& positions)
{
    return QMLP_CALL("combine_forward", combineForward).call(rows, weights, order, positions);
}
Tensor expertLinear(const Tensor& input, const Tensor& weight, const Tensor& offsets, const OptTensor& bias)
{
    return QMLP_CALL("expert_linear_forward", expertLinearForward).call(input, weight, offsets, bias);
}
