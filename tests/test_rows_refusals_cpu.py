"""What the registered operators on feature rows refuse, as far as it shows on meta tensors: the checks are those of the CUDA kernels."""
import pytest
import torch


@pytest.fixture(scope="module")
def error():
    import qmlp  # noqa: F401
    from qmlp._capi import QmlpError
    return QmlpError


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_layer_norm_stats(error):
    """the adjoint reads a mean and a deviation per row: statistics of another size, type or layout are refused"""
    adjoint = torch.ops.qmlp_b200.layer_norm_adjoint
    x = meta(6, 5, 8)
    assert adjoint(x, x, None, None, meta(2, 30), True, False, False)[0].shape == x.shape
    for stats in (meta(2, 29), meta(60), meta(30, 2), meta(2, 30, dtype=torch.float16), meta(30, 2).t(), meta(2, 0)):
        with pytest.raises(error, match="stats"):
            adjoint(x, x, None, None, stats, True, False, False)


def test_parameters_of_other_dimensions(error):
    """a weight or bias of more dimensions than a view holds, or of none (which is not "no parameter"), or of another width"""
    import qmlp
    x, h = meta(4, 8), meta(4, 8, dtype=torch.float16)
    for wrong in (meta(1, 1, 8), meta(1, 8), meta(1, 1, 1, 1, 1, 8), meta(), meta(7)):
        for weight, bias in ((wrong, None), (None, wrong), (meta(8), wrong)):
            with pytest.raises(error, match="wrong dimension|number of channels"):
                qmlp.layer_norm(x, weight, bias)
            with pytest.raises(error, match="wrong dimension|number of channels"):
                torch.ops.qmlp_b200.layer_norm_adjoint(x, x, weight, bias, meta(2, 4), True, True, True)
    matrices, offsets = meta(3, 5, 8, dtype=torch.float16), meta(4, dtype=torch.int32)
    assert qmlp.expert_linear(h, matrices, offsets, meta(3, 5, dtype=torch.float16)).shape == (4, 5)
    for wrong in (meta(), meta(5), meta(1, 3, 5), meta(3, 6)):
        with pytest.raises(error, match="bias"):
            qmlp.expert_linear(h, matrices, offsets, wrong.half())


def test_no_channels(error):
    """rows without a channel, and a tensor without a dimension, are an error and no division by zero (in a process of its own)"""
    import os
    import subprocess
    import sys
    code = """
import torch, qmlp
from qmlp._capi import QmlpError
ops = torch.ops.qmlp_b200
x, s = torch.empty((5, 0), device="meta"), torch.empty((), device="meta")
h, w = x.half(), torch.empty((2, 3, 0), dtype=torch.float16, device="meta")
o = torch.empty(3, dtype=torch.int32, device="meta")
calls = [lambda: qmlp.layer_norm(x), lambda: qmlp.layer_norm(s), lambda: ops.layer_norm_adjoint(x, x, None, None, torch.empty((2, 5), device="meta"), True, False, False),
         lambda: qmlp.expert_linear(h, w, o), lambda: ops.expert_linear_adjoint(h, torch.empty((5, 3), device="meta").half(), w, o, True, True, False)]
for call in calls:
    try:
        call()
    except QmlpError as e:
        assert "at least one" in str(e), e
    else:
        raise AssertionError("not refused")
print("fine")
"""
    package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "quick-mlp_b200")
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": package}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, (done.returncode, done.stderr[-2000:])


def test_forward_mode(error):
    """The operators have no forward-mode formula: a tangent is refused, whether or not a gradient is asked for, and never dropped."""
    import torch.autograd.forward_ad as fwad
    import qmlp
    half = torch.float16
    tokens, ints = meta(5, dtype=torch.int64), meta(12, dtype=torch.int32)
    positions, offsets = meta(6, 2, dtype=torch.int32), meta(4, dtype=torch.int32)
    r = qmlp.Routing(meta(6, 2), positions, ints, positions, offsets)
    ops = torch.ops.qmlp_b200
    calls = [   # a call of its differentiable arguments, and these
        (lambda x, w, b: qmlp.layer_norm(x, w, b), [meta(6, 8), meta(8), meta(8)]),
        (lambda t: qmlp.embedding(tokens, t), [meta(9, 8)]),
        (lambda z: qmlp.route(z, 2).weights, [meta(6, 3)]),
        (lambda x: qmlp.dispatch(x, r), [meta(6, 8)]),
        (lambda y, w: qmlp.combine(y, r._replace(weights=w)), [meta(12, 8), meta(6, 2)]),
        (lambda x, w, b: qmlp.expert_linear(x, w, offsets, b), [meta(12, 8, dtype=half), meta(3, 4, 8, dtype=half), meta(3, 4, dtype=half)]),
        (lambda x, g: ops.layer_norm_adjoint(x, g, None, None, meta(2, 6), True, False, False)[0], [meta(6, 8), meta(6, 8)]),
        (lambda g: ops.embedding_adjoint(tokens, g, 9, 1.0), [meta(5, 8)]),
        (lambda z, w, g: ops.route_adjoint(z, True, w, positions, g), [meta(6, 3), meta(6, 2), meta(6, 2)]),
        (lambda g: ops.dispatch_adjoint(g, positions), [meta(12, 8)]),
        (lambda y, g, w: ops.combine_adjoint(y, g, w, ints, positions, True, True)[0], [meta(12, 8), meta(6, 8), meta(6, 2)]),
        (lambda x, g, w: ops.expert_linear_adjoint(x, g, w, offsets, True, True, True)[0], [meta(12, 8, dtype=half), meta(12, 4, dtype=half), meta(3, 4, 8, dtype=half)]),
    ]
    for n, (call, args) in enumerate(calls):
        call(*args)
        for i, a in enumerate(args):
            for leaf in (a, a.clone().requires_grad_()):
                with fwad.dual_level(), pytest.raises(error, match="forward-mode"):
                    call(*args[:i], fwad.make_dual(leaf, torch.empty_like(a)), *args[i + 1:])
                    print("not refused:", n, i)
            with fwad.dual_level(), torch.no_grad(), pytest.raises(error, match="forward-mode"):
                call(*args[:i], fwad.make_dual(a, torch.empty_like(a)), *args[i + 1:])
        with pytest.raises(error, match="forward-mode"):
            torch.func.jvp(call, tuple(args), tuple(torch.empty_like(a) for a in args))


def test_functions_are_traceable():
    """torch.compile takes the functions and FusedExperts' layer whole, with their gradients: the registered operators stand in the graph"""
    import qmlp
    half = torch.float16
    seen = []

    def backend(graph, inputs):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    def model(tokens, table, w, b, router, weight, bias):
        x = qmlp.layer_norm(qmlp.embedding(tokens, table, 2.0), w, b)
        r = qmlp.route(x @ router, 2)
        return qmlp.combine(qmlp.expert_linear(qmlp.dispatch(x.half(), r), weight, r.offsets, bias), r)
    args = [meta(30, dtype=torch.int64), meta(9, 16), meta(16), meta(16), meta(16, 6), meta(6, 8, 16, dtype=half), meta(6, 8, dtype=half)]
    leaves = [a.requires_grad_() if a.is_floating_point() else a for a in args]
    torch._dynamo.reset()
    y = torch.compile(model, fullgraph=True, backend=backend)(*leaves)
    assert y.shape == (30, 8) and y.dtype == half
    for name in ("layer_norm", "embedding", "route", "dispatch", "combine", "expert_linear"):
        assert any(f"qmlp_b200.{name}_forward" in t for t in seen), (name, seen)
    y = torch.compile(model, fullgraph=True, backend="aot_eager")(*leaves)
    grads = torch.autograd.grad(y, leaves[1:], torch.empty_like(y))
    assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in leaves[1:]]
    layer = qmlp.FusedExperts(16, 32, 8, experts=4, dtype=torch.bfloat16, device="meta")
    assert torch.compile(layer, fullgraph=True, backend="aot_eager")(meta(5, 3, 16)).shape == (5, 3, 8)
    torch._dynamo.reset()


def test_first_call_is_traced():
    """torch.compile before anything has loaded the native call path (in a process of its own)"""
    import os
    import subprocess
    import sys
    code = """
import torch, qmlp
f = torch.compile(lambda x: qmlp.layer_norm(x) * 2, fullgraph=True, backend="aot_eager")
assert f(torch.empty((4, 8), device="meta", requires_grad=True)).shape == (4, 8)
print("fine")
"""
    package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "quick-mlp_b200")
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": package}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, (done.returncode, done.stderr[-2000:])
