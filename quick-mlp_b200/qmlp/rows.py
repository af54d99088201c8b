"""Operators on feature rows, for what stands between an encoding and a network or around several networks: layer norm, lookup of
latent codes, routing of rows to experts, matrix products grouped by expert.

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
from . import ops  # noqa: F401  (registers torch.ops.qmlp_b200.*)


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


class FusedExperts(torch.nn.Module):
    """A layer of experts: a router picks k of them for every row, each is a two-layer network with an activation of the
    package between its layers, and their outputs are added up with the router's weights.

    Parameters are kept in `weight_dtype` and cast to `dtype` (the type of the products) per call, like FusedNetwork's."""

    def __init__(self, channels_in: int, channels_hidden: int, channels_out: int, experts: int, k: int = 2, activation: str = "relu",
                 normalize: bool = True, weight_dtype=torch.float32, dtype=torch.float16, device="cuda"):
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

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape, x = x.shape, x.reshape(-1, x.shape[-1])
        routing = route(torch.nn.functional.linear(x.float(), self.router.float()), self.k, self.normalize)
        h = dispatch(x.to(self.dtype), routing)
        h = expert_linear(h, self.weight1.to(self.dtype), routing.offsets, self.bias1.to(self.dtype))
        h = expert_linear(self.activation(h), self.weight2.to(self.dtype), routing.offsets, self.bias2.to(self.dtype))
        y = combine(h, routing)
        return y.reshape(*shape[:-1], y.shape[-1])

    def extra_repr(self):
        e, hidden, n_in = self.weight1.shape
        return f"{n_in} -> {hidden} -> {self.weight2.shape[1]}, experts={e}, k={self.k}"
