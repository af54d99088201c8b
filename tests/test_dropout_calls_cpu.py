"""Which call of a dropout layer drops what, as far as it goes without a GPU: calls that are recomputed in a backward pass."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


class Block(torch.nn.Module):
    def __init__(self, dropout):
        super().__init__()
        self.linear, self.dropout = torch.nn.Linear(16, 16, device="meta"), dropout

    def forward(self, x):
        return self.dropout(self.linear(x)).relu()


def test_step_is_not_recomputed(qmlp):
    """a count of calls is read and advanced, but not in a backward pass, whatever recomputes it there"""
    from qmlp import ops
    from qmlp._capi import QmlpError
    step = torch.tensor([4])
    assert int(ops.dropout_step(step)) == 4 and int(torch.ops.qmlp_b200.dropout_step(step)) == 5 and int(step) == 6

    class Advance(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, call):
            ctx.call = call
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            ctx.call(step)
            return g, None
    x = torch.ones(3, requires_grad=True)
    for call in (ops.dropout_step, torch.ops.qmlp_b200.dropout_step):
        y = Advance.apply(x, call).sum()
        with pytest.raises(QmlpError, match="recomputed"):
            y.backward()
    assert int(step) == 6


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("compiled", [False, True])
def test_checkpointed_with_a_seed(qmlp, reentrant, compiled):
    """a layer with a seed under torch.utils.checkpoint: an error instead of the gradient of other elements"""
    torch._dynamo.reset()
    block = Block(qmlp.FusedDropout(0.3, seed=5, device="meta"))
    call = torch.compile(block, fullgraph=True, backend="aot_eager") if compiled else block
    x = meta(6, 16).requires_grad_()
    call(x).sum().backward()
    y = checkpoint(call, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="recomputed"):
        y.sum().backward()
    experts = qmlp.FusedExperts(16, 32, 8, experts=4, device="meta", dropout=0.2, seed=1)
    y = checkpoint(experts, meta(5, 16).requires_grad_(), use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="recomputed"):
        y.sum().backward()
    torch._dynamo.reset()


def test_checkpoint_in_a_compiled_call(qmlp):
    torch._dynamo.reset()
    block = Block(qmlp.FusedDropout(0.3, seed=5, device="meta"))
    call = torch.compile(lambda x: checkpoint(block, x, use_reentrant=False), fullgraph=True, backend="aot_eager")
    with pytest.raises(RuntimeError, match="recomputed"):
        call(meta(6, 16).requires_grad_()).sum().backward()
    torch._dynamo.reset()


def test_layers_without_a_seed(qmlp, monkeypatch):
    """every call of every layer takes a number of its own from torch's generator, which repeats it; a seed that is given stays what it is, 0 too"""
    seen = []
    real = torch.randint
    monkeypatch.setattr(torch, "randint", lambda high, size, device: real(high, size))      # (numbers, where meta tensors have none)
    monkeypatch.setattr(qmlp.rows, "dropout", lambda x, p, seed, offset, residual, step: seen.append((seed, offset, int(step))) or x)
    layers = [qmlp.FusedDropout(0.5, device="meta") for _ in range(2)] + [qmlp.FusedExperts(16, 32, 8, experts=4, device="meta", dropout=0.5).dropout]

    def run():
        seen.clear()
        torch.manual_seed(9)
        for _ in range(3):
            for layer in layers:
                layer(meta(4, 8))
        return list(seen)
    first = run()
    assert len(set(first)) == 9 and run() == first
    seen.clear()
    torch.manual_seed(10)
    layers[0](meta(4, 8))
    assert seen[0] != first[0]
    for seed in (0, 7):
        counted = qmlp.FusedDropout(0.5, seed, device="cpu")
        seen.clear()
        for _ in range(3):
            counted(meta(4, 8))
        assert seen == [(seed, 0, i) for i in range(3)]


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("compiled", [False, True])
def test_checkpointed_without_a_seed(qmlp, reentrant, compiled):
    torch._dynamo.reset()
    block = Block(qmlp.FusedDropout(0.3, device="meta"))
    call = torch.compile(block, fullgraph=True, backend="aot_eager") if compiled else block
    x = meta(6, 16).requires_grad_()
    checkpoint(call, x, use_reentrant=reentrant).sum().backward()
    assert x.grad.shape == x.shape
    torch._dynamo.reset()


@pytest.mark.parametrize("dropout", [-0.1, 1.5, float("nan")])
def test_experts_refuse_what_is_no_probability(qmlp, dropout):
    with pytest.raises(ValueError, match="between 0 and 1"):
        qmlp.FusedExperts(16, 32, 8, experts=4, device="meta", dropout=dropout)
