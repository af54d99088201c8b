"""Operators on feature rows, for what stands between an encoding and a network or around several networks: layer norm, lookup of
latent codes, routing of rows to experts, matrix products grouped by expert, dropout, matrices in 4 bits and products with them.

The reference leaves these to PyTorch. Here they are kernels of the library behind registered operators
(torch.ops.qmlp_b200.layer_norm_forward, ... in qmlp/ops.py), differentiable once. Features are float32, float16 or
bfloat16 tensors (..., channels); sums are float32, results have the features' type. Results are the same every run.

The functions call the native call path, which goes through the dispatcher without the interpreter's detour. While torch.compile traces, which
cannot look into it, they call the registered operators themselves.
"""
from typing import NamedTuple, Optional

import torch
from torch.compiler import assume_constant_result, is_compiling

from . import _capi
from . import ops  # (registers torch.ops.qmlp_b200.*)


@assume_constant_result
def _loaded():
    """loads the kernels behind the registered operators, while torch.compile traces"""
    _capi.calls()
    return True


class Routing(NamedTuple):
    """Which rows go to which experts. Slot s = row * k + j is the j-th choice of a row."""
    weights: torch.Tensor     # (rows, k) float32: weight of a choice, 0 in a slot without an expert; differentiable
    experts: torch.Tensor     # (rows, k) int32: expert, -1 in a slot without one
    order: torch.Tensor       # (rows * k) int32: slots, expert by expert, ascending within one; -1 behind the last expert's
    positions: torch.Tensor   # (rows, k) int32: place of a slot in `order`, -1 for none
    offsets: torch.Tensor     # (experts + 1) int32: where the slots of an expert begin in `order`


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension. weight, bias: float32 or x's type."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.layer_norm_forward(x, weight, bias, eps)[0]
    return _capi.calls().layer_norm(x, weight, bias, eps)


def embedding(tokens: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * table[tokens] for int32 or int64 tokens of any shape. A token outside the table (-1, say) is masked: its row
    is zeros and it contributes to no gradient. The table's gradient sums the sorted tokens' rows in float32, in their order."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.embedding_forward(tokens, table, scale)
    return _capi.calls().embedding(tokens, table, scale)


def route(logits: torch.Tensor, k: int, normalize: bool = True) -> Routing:
    """The k (at most 32) experts with the largest logits of every row of (rows, experts <= 1024), ties to the lowest index.
    Weights are a softmax over the chosen experts (normalize) or over all of the row. An expert with logit -inf is never
    chosen: a row with fewer than k others has slots without an expert."""
    if is_compiling() and _loaded():
        return Routing(*torch.ops.qmlp_b200.route_forward(logits, k, normalize))
    return Routing(*_capi.calls().route(logits, k, normalize))


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Feature rows (rows, channels) -> (rows * k, channels) in the experts' order; zeros behind the last expert's rows."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.dispatch_forward(x, routing.order, routing.positions)
    return _capi.calls().dispatch(x, routing.order, routing.positions)


def combine(rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Rows in the experts' order -> (rows, channels): the weighted sum of each row's slots."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.combine_forward(rows, routing.weights, routing.order, routing.positions)
    return _capi.calls().combine(rows, routing.weights, routing.order, routing.positions)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = weight[e] @ x[r] + bias[e] for the rows r in [offsets[e], offsets[e + 1]) of expert e; rows of no expert are zeros.

    x: (rows, channels in), weight: (experts <= 2048, channels out, channels in), bias: (experts, channels out), all float16 or
    all bfloat16; offsets: (experts + 1) ascending int32 on the device (Routing.offsets)."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.expert_linear_forward(x, weight, offsets, bias)
    return _capi.calls().expert_linear(x, weight, offsets, bias)


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0, residual: Optional[torch.Tensor] = None, step: Optional[torch.Tensor] = None) -> torch.Tensor:
    """residual + x / (1 - p) where an element is kept, residual (or 0) where it is dropped, with probability p (in units of 2^-16).

    Which are dropped follows from seed and offset (int64) and an element's place: 16 bits of Philox4x32-10 with the key `seed` and the counter
    (element // 8, offset + step). No mask is stored; another call with the same numbers drops the same. step: an int64 tensor of one element
    on the device that is added to the offset when the kernel runs, so that a captured graph draws new numbers when its program advances it."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.dropout_forward(x, residual, p, seed, offset, step)
    return _capi.calls().dropout(x, p, seed, offset, residual, step)


class MXTensor(NamedTuple):
    """A matrix (rows, channels) or matrices (matrices, rows, channels) in microscaled 4-bit floating point (MXFP4): 32 channels of a row share a power of two,
    elements are e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign)."""
    codes: torch.Tensor     # (..., rows, 16 * ceil(channels / 32)) uint8: two elements a byte, the first in the low bits, zeros behind the last channel
    scales: torch.Tensor    # (..., ceil(rows / 128), ceil(channels / 128), 32, 4, 4) uint8: [t, c, i, q, j] is the exponent + 127 (255: NaN) of row
    channels: int           # 128 t + 32 q + i and of the channels from 128 c + 32 j on, zero where there is no such block


def mx_quantize(x: torch.Tensor) -> MXTensor:
    """x (rows, channels) or (matrices, rows, channels) in 4 bits. A block's power of two is floor(log2(largest magnitude)) - 2, elements are rounded to the
    nearest (ties to the even code, at most 6 in magnitude); a block with an infinity or NaN becomes NaN. No gradient."""
    if is_compiling() and _loaded():
        return MXTensor(*torch.ops.qmlp_b200.mx_quantize(x), x.shape[-1])
    return MXTensor(*_capi.calls().mx_quantize(x), x.shape[-1])


def mx_dequantize(q: MXTensor, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values of q in float32, float16 or bfloat16 (exact within the type's range, which of the first and the last covers what mx_quantize gives)."""
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.mx_dequantize(q.codes, q.scales, q.channels, dtype)
    return _capi.calls().mx_dequantize(q.codes, q.scales, q.channels, dtype)


def mx_linear(x: torch.Tensor, weight: MXTensor, offsets: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows times 4-bit matrices, as expert_linear: y[r] = weight[e] @ q(x[r]) + bias[e] for the rows r in [offsets[e], offsets[e + 1]), with q(x[r]) the row
    in 4 bits too (mx_quantize); rows of no expert are zeros. A single matrix (channels out, channels in) takes no offsets and a bias (channels out).

    x: (..., channels in) float16 or bfloat16, bias of the same type. Gradients of x and bias: the quantisation of x counts as the identity, the weights are
    constants, exact over the whole range that mx_quantize gives (float16 gradients of matrices whose blocks lie more than 2^26 apart take many times as long)."""
    if x.shape[-1:] != (weight.channels,):
        raise _capi.QmlpError(f"x must have the weight's {weight.channels} channels")
    if is_compiling() and _loaded():
        return torch.ops.qmlp_b200.mx_linear_forward(x, weight.codes, weight.scales, offsets, bias)
    return _capi.calls().mx_linear(x, weight.codes, weight.scales, offsets, bias)


class FusedLayerNorm(torch.nn.Module):
    """Layer norm over the last dimension with float32 parameters, for features of any of the three types."""

    def __init__(self, channels: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device="cuda"):
        super().__init__()
        self.channels, self.eps = channels, eps
        self.weight = torch.nn.Parameter(torch.ones(channels, device=device)) if elementwise_affine else None
        self.bias = torch.nn.Parameter(torch.zeros(channels, device=device)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.channels}, eps={self.eps}"


class FusedEmbedding(torch.nn.Module):
    """A table of latent codes, one row per token (an image, a frame, a word)."""

    def __init__(self, rows: int, channels: int, scale: float = 1.0, dtype=torch.float32, device="cuda"):
        super().__init__()
        self.scale = scale
        self.table = torch.nn.Parameter(torch.empty((rows, channels), dtype=dtype, device=device))
        torch.nn.init.normal_(self.table, std=0.01)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.table, self.scale)

    def extra_repr(self):
        return f"{tuple(self.table.shape)}, scale={self.scale}"


class FusedDropout(torch.nn.Module):
    """Dropout in training, nothing but the residual's addition in evaluation.

    Without a seed every call takes its numbers from a draw of torch's generator of x's device, as torch's own dropout: layers drop different elements, a
    captured step other ones every time it is replayed, torch.manual_seed repeats them (ranks that are to differ seed differently), and a call
    that is recomputed in a backward pass (activation checkpointing, which restores the generator) drops the same ones.

    With a seed the numbers follow from it and from `step`, which counts the calls on the device: layers of equal seeds drop equal elements, a captured step counts on
    in every replay, and a state_dict that is loaded goes on where it was saved. A recomputed call is refused then: the count does not say which call it repeats."""

    def __init__(self, p: float, seed: Optional[int] = None, device="cuda"):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError("p must be between 0 and 1")
        self.p, self.seed = p, seed
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64, device=device))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training:
            return x if residual is None else x + residual
        if self.seed is None:
            return dropout(x, self.p, 0, 0, residual, torch.randint(2 ** 63 - 1, (1,), device=x.device))
        step = (torch.ops.qmlp_b200 if is_compiling() else ops).dropout_step(self.step)      # what the gradient's call reads too
        return dropout(x, self.p, self.seed, 0, residual, step)

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"


class FusedExperts(torch.nn.Module):
    """A layer of experts: a router picks k of them for every row, each is a two-layer network with an activation of the
    package between its layers, and their outputs are added up with the router's weights.

    Parameters are kept in `weight_dtype` and cast to `dtype` (the type of the products) per call, like FusedNetwork's.
    dropout: share of the hidden channels dropped in training (behind the activation), with or without a `seed` as FusedDropout.
    quantized() gives the layer with its matrices in 4 bits."""

    def __init__(self, channels_in: int, channels_hidden: int, channels_out: int, experts: int, k: int = 2, activation: str = "relu",
                 normalize: bool = True, weight_dtype=torch.float32, dtype=torch.float16, device="cuda", dropout: float = 0.0, seed: Optional[int] = None):
        super().__init__()
        from .activation import FusedActivation
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("the products are computed in float16 or bfloat16")
        self.k, self.normalize, self.dtype = k, normalize, dtype
        # the package's activations compute in half
        self.activation = FusedActivation(activation) if dtype == torch.float16 else torch.nn.ReLU()
        if dtype != torch.float16 and activation != "relu":
            raise ValueError("activations other than relu need dtype=torch.float16")

        def uniform(*shape, fan_in):
            return torch.nn.Parameter(torch.empty(shape, dtype=weight_dtype, device=device).uniform_(-1, 1).mul_(fan_in ** -0.5))
        self.router = uniform(experts, channels_in, fan_in=channels_in)
        self.weight1 = uniform(experts, channels_hidden, channels_in, fan_in=channels_in)
        self.bias1 = torch.nn.Parameter(torch.zeros((experts, channels_hidden), dtype=weight_dtype, device=device))
        self.weight2 = uniform(experts, channels_out, channels_hidden, fan_in=channels_hidden)
        self.bias2 = torch.nn.Parameter(torch.zeros((experts, channels_out), dtype=weight_dtype, device=device))
        self.dropout = FusedDropout(dropout, seed, device) if dropout != 0 else None      # (which refuses what is no probability)

    def quantized(self) -> "QuantizedExperts":
        """A copy whose matrices are kept and multiplied in 4 bits, for serving."""
        return QuantizedExperts(self)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape, x = x.shape, x.reshape(-1, x.shape[-1])
        routing = route(torch.nn.functional.linear(x.float(), self.router.float()), self.k, self.normalize)
        h = dispatch(x.to(self.dtype), routing)
        h = expert_linear(h, self.weight1.to(self.dtype), routing.offsets, self.bias1.to(self.dtype))
        h = self.activation(h)
        if self.dropout is not None:
            h = self.dropout(h)
        h = expert_linear(h, self.weight2.to(self.dtype), routing.offsets, self.bias2.to(self.dtype))
        y = combine(h, routing)
        return y.reshape(*shape[:-1], y.shape[-1])

    def extra_repr(self):
        e, hidden, n_in = self.weight1.shape
        return f"{n_in} -> {hidden} -> {self.weight2.shape[1]}, experts={e}, k={self.k}"


class QuantizedExperts(torch.nn.Module):
    """A layer of experts (FusedExperts) with its matrices in 4 bits; the rows of both products are quantised in their calls. Nothing of it is trained; gradients
    of the rows pass through (mx_linear), for what is in front of it.
    The router and the biases are cast per call, like FusedExperts', so that a model may be cast as a whole."""

    def __init__(self, layer: FusedExperts):
        super().__init__()
        self.k, self.normalize, self.dtype, self.activation = layer.k, layer.normalize, layer.dtype, layer.activation
        self.channels_in, self.channels_hidden = layer.weight1.shape[2], layer.weight2.shape[2]
        with torch.no_grad():
            tensors = {"router": layer.router.float(), "bias1": layer.bias1.to(self.dtype), "bias2": layer.bias2.to(self.dtype)}
            tensors = {name: t.detach().clone() for name, t in tensors.items()}      # (of the type it should be, `to` gives the parameter itself)
            for name, weight in (("1", layer.weight1), ("2", layer.weight2)):
                weight = weight.detach()
                tensors["codes" + name], tensors["scales" + name], _ = mx_quantize(weight.float() if weight.dtype == torch.float64 else weight)
        for name, t in tensors.items():
            self.register_buffer(name, t)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape, x = x.shape, x.reshape(-1, x.shape[-1])
        routing = route(torch.nn.functional.linear(x.float(), self.router.float()), self.k, self.normalize)
        h = dispatch(x.to(self.dtype), routing)
        h = self.activation(mx_linear(h, MXTensor(self.codes1, self.scales1, self.channels_in), routing.offsets, self.bias1.to(self.dtype)))
        h = mx_linear(h, MXTensor(self.codes2, self.scales2, self.channels_hidden), routing.offsets, self.bias2.to(self.dtype))
        y = combine(h, routing)
        return y.reshape(*shape[:-1], y.shape[-1])

    def extra_repr(self):
        return f"{self.channels_in} -> {self.channels_hidden} -> {self.bias2.shape[1]}, experts={self.bias1.shape[0]}, k={self.k}, 4 bits"
