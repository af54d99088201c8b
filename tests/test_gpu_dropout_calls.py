"""Which elements the calls of dropout layers drop: layers side by side, calls that are recomputed in a backward pass, captured ones."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def test_layers_differ(qmlp):
    """layers without a seed drop independently of one another and of their calls before: the share that two drop together is p^2, within five deviations"""
    torch.manual_seed(1)
    n, p = 1 << 20, 0.25
    x = torch.ones((n // 64, 64), device="cuda")
    layers = [qmlp.FusedDropout(p) for _ in range(2)]
    dropped = [layer(x) == 0 for layer in layers for _ in range(2)]
    for i, a in enumerate(dropped):
        assert abs(a.double().mean().item() - p) < 5 * (p * (1 - p) / n) ** 0.5
        for b in dropped[:i]:
            assert abs((a & b).double().mean().item() - p * p) < 5 * (p * p * (1 - p * p) / n) ** 0.5
    torch.manual_seed(1)
    assert all(torch.equal(a, layer(x) == 0) for a, layer in zip(dropped, [layers[0], layers[0], layers[1], layers[1]]))
    a, b = qmlp.FusedDropout(p, seed=4), qmlp.FusedDropout(p, seed=4)
    assert torch.equal(a(x), b(x)) and torch.equal(a(x), qmlp.dropout(x, p, 4, 1))


class Model(torch.nn.Module):
    """layers with dropout, one of them used twice"""

    def __init__(self, qmlp):
        super().__init__()
        self.first, self.second = (qmlp.FusedExperts(32, 64, 32, experts=4, k=2, dropout=0.5) for _ in range(2))
        self.dropout = qmlp.FusedDropout(0.3)

    def forward(self, x, call):
        x = call(self.first, x)
        x = call(lambda v: self.dropout(v.half(), v.half()).float(), x)
        x = call(self.second, x).float()
        return call(lambda v: self.dropout(self.first(v)), x)


@pytest.mark.parametrize("reentrant", [True, False])
def test_checkpointed(qmlp, reentrant):
    """output and gradients with and without checkpoints are the same bits, and so is what comes after"""
    torch.manual_seed(2)
    model = Model(qmlp)
    x, g = rand(3, (300, 32)), rand(4, (300, 32), torch.float16)

    def run(call):
        torch.manual_seed(5)
        leaf, out = x.clone().requires_grad_(), []
        for _ in range(2):
            y = model(leaf, call)
            y.backward(g)
            out += [y.detach(), leaf.grad.clone(), *(p.grad.clone() for p in model.parameters())]
            leaf.grad = None
            model.zero_grad()
        return out + [model(x, lambda f, v: f(v)).detach()]
    want = run(lambda f, v: f(v))
    got = run(lambda f, v: checkpoint(f, v, use_reentrant=reentrant))
    assert len(got) == len(want) and all(torch.equal(a, e) for a, e in zip(got, want))
    assert not torch.equal(want[0], want[len(want) // 2])


def test_compiled(qmlp):
    """traced whole, checkpointed or not: the gradient is that of the elements that were dropped"""
    torch._dynamo.reset()
    layer = qmlp.FusedDropout(0.4)
    x = torch.ones((200, 24), device="cuda")
    for call in (torch.compile(layer, fullgraph=True, backend="aot_eager"), torch.compile(lambda v: checkpoint(layer, v, use_reentrant=False), fullgraph=True, backend="aot_eager"),
                 lambda v: checkpoint(torch.compile(layer, fullgraph=True, backend="aot_eager"), v, use_reentrant=False)):
        leaf = x.clone().requires_grad_()
        y, again = call(leaf), call(leaf)
        assert not torch.equal(y, again) and 0.2 < (y == 0).double().mean().item() < 0.6
        for out in (y, again):
            assert torch.equal(torch.autograd.grad(out, leaf, x)[0], out)
    torch._dynamo.reset()


def test_captured(qmlp):
    """a step in a graph, without a seed: every replay drops other elements, and its gradient the same ones"""
    layer = qmlp.FusedDropout(0.5)
    leaf = torch.ones((100, 64), device="cuda").requires_grad_()

    def step():
        y = layer(leaf)
        return y.detach(), torch.autograd.grad(y, leaf, torch.ones_like(y))[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
    seen = []
    for _ in range(3):
        graph.replay()
        assert torch.equal(y, dx)
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_compiled_with_a_seed(qmlp):
    """compiled, a layer with a seed counts on: the elements of the eager calls, and their gradients"""
    torch._dynamo.reset()
    layer, x, r = qmlp.FusedDropout(0.4, seed=3), rand(6, (200, 24)), rand(7, (200, 24))
    compiled = torch.compile(layer, fullgraph=True, backend="aot_eager")
    outs = []
    for i, call in enumerate((compiled, layer, compiled, compiled)):
        leaf = x.clone().requires_grad_()
        y = call(leaf, r)
        assert torch.equal(y, qmlp.dropout(x, 0.4, 3, i, residual=r)) and int(layer.step) == i + 1
        outs.append((y, leaf, i))
    for y, leaf, i in outs:
        assert torch.equal(torch.autograd.grad(y, leaf, r)[0], qmlp.dropout(r, 0.4, 3, i))
    torch._dynamo.reset()
