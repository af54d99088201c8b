"""Dropout and 4-bit layers as they are used: in a layer of experts that is trained, captured and then served in 4 bits, next to the other operators on feature rows;
calls of the C ABI with too little scratch memory."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(dtype)


def test_dropout_module(qmlp):
    """a call of the function with the count of calls; nothing in evaluation; the count is saved and loaded"""
    layer, x, r = qmlp.FusedDropout(0.3, seed=7), rand(1, (50, 40)), rand(2, (50, 40))
    for i in range(3):
        assert torch.equal(layer(x, r), qmlp.dropout(x, 0.3, 7, i, residual=r))
    other = qmlp.FusedDropout(0.3, seed=7)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), layer(x)) and torch.equal(layer(x), qmlp.dropout(x, 0.3, 7, 4))
    leaf = x.clone().requires_grad_()
    y = layer(leaf)
    layer(leaf)      # (a later call leaves the earlier one's gradient alone)
    assert torch.equal(torch.autograd.grad(y, leaf, r)[0], qmlp.dropout(r, 0.3, 7, 5))
    layer.eval()
    assert layer(x) is x and torch.equal(layer(x, r), x + r) and int(layer.step) == 7


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["half", "bfloat16"])
def test_experts(qmlp, dtype):
    """a layer of experts with dropout, and its copy in 4 bits: the operators one after the other, with their gradients; without dropout the layer is as it was"""
    torch.manual_seed(3)
    layer = qmlp.FusedExperts(48, 100, 24, experts=6, k=2, dtype=dtype, dropout=0.25, seed=11)
    plain = qmlp.FusedExperts(48, 100, 24, experts=6, k=2, dtype=dtype)
    plain.load_state_dict({k: v for k, v in layer.state_dict().items() if not k.startswith("dropout")})
    x, g = rand(4, (700, 48)), rand(5, (700, 24), dtype)

    def by_hand(x, first, second, drop):
        r = qmlp.route(torch.nn.functional.linear(x.float(), layer.router), 2)
        h = layer.activation(first(qmlp.dispatch(x.to(dtype), r), r.offsets))
        return qmlp.combine(second(drop(h), r.offsets), r)

    def product(weight, bias):
        return lambda h, o: qmlp.expert_linear(h, weight.to(dtype), o, bias.to(dtype))
    first, second = product(layer.weight1, layer.bias1), product(layer.weight2, layer.bias2)
    params = [layer.router, layer.weight1, layer.bias1, layer.weight2, layer.bias2]
    for call in range(2):
        leaves = [x.clone().requires_grad_() for _ in range(2)]
        y = layer(leaves[0])
        want = by_hand(leaves[1], first, second, lambda h: qmlp.dropout(h, 0.25, 11, call))
        assert torch.equal(y, want)
        got, grads = torch.autograd.grad(y, [leaves[0], *params], g), torch.autograd.grad(want, [leaves[1], *params], g)
        assert all(torch.equal(a, e) for a, e in zip(got, grads))
    layer.eval()
    with torch.no_grad():
        assert torch.equal(layer(x), plain(x)) and torch.equal(plain(x), by_hand(x, first, second, lambda h: h))

    served = layer.quantized()
    q1, q2 = qmlp.mx_quantize(layer.weight1.detach()), qmlp.mx_quantize(layer.weight2.detach())
    q_first, q_second = (lambda h, o: qmlp.mx_linear(h, q1, o, layer.bias1.detach().to(dtype))), (lambda h, o: qmlp.mx_linear(h, q2, o, layer.bias2.detach().to(dtype)))
    leaves = [x.clone().requires_grad_() for _ in range(2)]
    y, want = served(leaves[0]), by_hand(leaves[1], q_first, q_second, lambda h: h)
    assert torch.equal(y, want) and torch.equal(torch.autograd.grad(y, leaves[0], g)[0], torch.autograd.grad(want, leaves[1], g)[0])
    again = qmlp.FusedExperts(48, 100, 24, experts=6, k=2, dtype=dtype).quantized()
    again.load_state_dict(served.state_dict())
    with torch.no_grad():
        for rows in (1, 3, 64, 700):      # single rows, small calls, larger ones
            assert torch.equal(again(x[:rows]), served(x[:rows]))
            assert torch.allclose(served(x[:rows]).float(), y[:rows].detach().float(), rtol=2.0 ** -6, atol=2.0 ** -6)
        exact = qmlp.FusedExperts(48, 100, 24, experts=6, k=2, dtype=dtype, weight_dtype=dtype)      # (parameters of the products' type)
        copied = exact.quantized()
        before = copied(x)
        for p in exact.parameters():
            p.add_(1)
        assert torch.equal(copied(x), before)


def test_training_step_captured(qmlp):
    """a training step in a graph: each replay drops other elements, those of the eager steps"""
    torch.manual_seed(5)
    layer = qmlp.FusedExperts(32, 64, 16, experts=4, k=2, dropout=0.5, seed=3)
    x, target = rand(6, (300, 32)), rand(7, (300, 16), torch.float16)

    def step():
        y = layer(x)
        return [y.detach(), *torch.autograd.grad(torch.nn.functional.mse_loss(y.float(), target.float()), list(layer.parameters()))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    layer.dropout.step.zero_()
    want = [step() for _ in range(3)]
    assert not torch.equal(want[0][0], want[1][0])
    layer.dropout.step.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    layer.dropout.step.zero_()
    for w in want:
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, w))


def test_compiled(qmlp):
    """traced by torch.compile: the results of the functions"""
    def model(x, r, w, b, step):
        q = qmlp.mx_quantize(w)
        return qmlp.mx_linear(qmlp.dropout(x, 0.3, 5, 2, residual=r, step=step), q, None, b) + qmlp.mx_dequantize(q, torch.float16).sum()
    x, r, w, b = (t.requires_grad_() for t in (rand(8, (200, 40), torch.float16), rand(9, (200, 40), torch.float16), rand(10, (24, 40)), rand(11, (24,), torch.float16)))
    step, g, results = torch.tensor([4], device="cuda"), rand(12, (200, 24), torch.float16), []
    for call in (model, torch.compile(model, fullgraph=True, backend="aot_eager")):
        y = call(x, r, w, b, step)
        results.append([y.detach(), *torch.autograd.grad(y, [x, r, b], g)])
    for a, e in zip(*results):
        assert torch.equal(a, e)


def test_example():
    """the example with dropout: it runs, its parameters get gradients, its copy in 4 bits answers"""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "images_by_experts.py")
    spec = importlib.util.spec_from_file_location("images_by_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    model = module.ImagesByExperts(3, dropout=0.1)
    x, image = torch.rand((500, 2), device="cuda"), torch.randint(3, (500,), device="cuda")
    model(x, image).sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters() if p.requires_grad)
    served = model.served()
    with torch.no_grad():
        assert torch.isfinite(served(x, image)).all() and isinstance(model.experts, type(module.qmlp.FusedExperts(4, 4, 4, 2)))
    said = []
    assert len(module.fit(images=2, points=512, steps=3, report=said.append, dropout=0.1)) == 3 and "4 bits" in said[-1]


def test_scratch(qmlp):
    """a product that needs scratch memory and gets too little, or off its alignment, is refused before a launch"""
    from qmlp import _capi
    lib = _capi.lib()
    x, y = rand(13, (5000, 2048), torch.float16), rand(14, (5000, 2048), torch.float16)
    q = qmlp.mx_quantize(rand(15, (2048, 2048)))
    m = _capi.Mx(matrices=1, rows=2048, channels=2048, codes=q.codes.data_ptr(), scales=q.scales.data_ptr())

    def view(t):
        v = _capi.Tensor(data=t.data_ptr(), precision=_capi.QMLP_HALF, ndim=2)
        v.sizes[0], v.sizes[1], v.strides[0], v.strides[1] = *t.shape, *t.stride()
        return C.byref(v)
    size, stream = C.c_size_t(), _capi.current_stream()
    for memory, flags, call in ((lib.qmlp_mx_linear_forward_memory, (), lambda p, n: lib.qmlp_mx_linear_forward(view(x), C.byref(m), None, None, view(y), stream, p, n)),
                                (lib.qmlp_mx_linear_adjoint_memory, (1,), lambda p, n: lib.qmlp_mx_linear_adjoint(view(y), C.byref(m), None, view(x), None, stream, p, n))):
        assert memory(view(x), C.byref(m), *flags, C.byref(size)) == 0 and size.value > 0
        scratch = torch.empty(size.value + 256, dtype=torch.uint8, device="cuda")
        for p, n in ((None, 0), (scratch.data_ptr(), size.value - 1), (scratch.data_ptr() + 16, size.value)):
            assert call(p, n) != 0 and "scratch memory" in lib.qmlp_last_error().decode()
        assert call(scratch.data_ptr(), size.value) == 0
    torch.cuda.synchronize()
