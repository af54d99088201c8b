"""The operators on feature rows as far as they go without a GPU: shapes, types and autograd graphs on meta tensors, and the argument
checks of the C ABI."""
import ctypes as C

import pytest


def _lib():
    from qmlp import _capi
    return _capi.lib()


def test_row_operators_on_meta_tensors():
    """Shapes, types and the autograd graph of the operators on feature rows, without a GPU: outputs and the gradients of every
    differentiable argument; a second differentiation fails."""
    import torch
    import qmlp
    half, meta = torch.float16, "meta"
    x = torch.empty((6, 10, 24), dtype=half, device=meta, requires_grad=True)
    w, b = torch.empty(24, device=meta, requires_grad=True), torch.empty(24, device=meta, requires_grad=True)
    y = qmlp.layer_norm(x, w, b)
    assert y.shape == x.shape and y.dtype == half
    grads = torch.autograd.grad(y, [x, w, b], torch.empty_like(y))
    assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in (x, w, b)]
    bias_only, = torch.autograd.grad(qmlp.layer_norm(x.detach(), None, b), [b], torch.empty_like(y))
    assert bias_only.shape == b.shape

    table = torch.empty((100, 24), device=meta, requires_grad=True)
    tokens = torch.empty((5, 7), dtype=torch.int64, device=meta)
    e = qmlp.embedding(tokens, table, 2.0)
    assert e.shape == (5, 7, 24) and torch.autograd.grad(e, table, torch.empty_like(e))[0].shape == table.shape

    logits = torch.empty((60, 8), dtype=half, device=meta, requires_grad=True)
    r = qmlp.route(logits, 2)
    assert (r.weights.shape, r.weights.dtype) == ((60, 2), torch.float32) and r.weights.requires_grad
    assert [tuple(t.shape) for t in (r.experts, r.order, r.positions, r.offsets)] == [(60, 2), (120,), (60, 2), (9,)]
    assert all(t.dtype == torch.int32 and not t.requires_grad for t in (r.experts, r.order, r.positions, r.offsets))
    rows = qmlp.dispatch(x.reshape(60, 24), r)
    weight = torch.empty((8, 40, 24), dtype=half, device=meta, requires_grad=True)
    bias = torch.empty((8, 40), dtype=half, device=meta, requires_grad=True)
    out = qmlp.combine(qmlp.expert_linear(rows, weight, r.offsets, bias), r)
    assert rows.shape == (120, 24) and out.shape == (60, 40) and out.dtype == half
    leaves = [x, logits, weight, bias]
    grads = torch.autograd.grad(out, leaves, torch.empty_like(out), create_graph=True)
    assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in leaves]
    with pytest.raises(RuntimeError, match="differentiable"):
        grads[2].sum().backward()


def test_row_operators_need_a_gpu():
    """Tensors of the CPU are refused with the package's error, not computed by something else."""
    import torch
    import qmlp
    from qmlp._capi import QmlpError
    x = torch.ones((4, 8))
    for call in (lambda: qmlp.layer_norm(x), lambda: qmlp.embedding(torch.zeros(3, dtype=torch.int64), x), lambda: qmlp.route(x, 2)):
        with pytest.raises(QmlpError, match="CUDA"):
            call()


def test_row_operator_refusals():
    """Argument checks of the operators on feature rows, which come before anything touches a device: types, sizes, strides, limits,
    scratch memory. The pointers are never followed."""
    from qmlp import _capi
    lib = _lib()
    here = C.create_string_buffer(4096)
    at = (C.addressof(here) + 255) // 256 * 256

    def matrix(rows, channels, precision=_capi.QMLP_HALF, strides=None, data=at):
        t = _capi.Tensor(data=data, precision=precision, ndim=2)
        t.sizes[0], t.sizes[1] = rows, channels
        t.strides[0], t.strides[1] = strides or (channels, 1)
        return C.byref(t)

    def vector(n, precision=_capi.QMLP_FLOAT, stride=1):
        t = _capi.Tensor(data=at, precision=precision, ndim=1)
        t.sizes[0], t.strides[0] = n, stride
        return C.byref(t)

    def routing(tokens=4, experts=8, chosen=2, **missing):
        r = _capi.Routing(tokens=tokens, num_experts=experts, chosen=chosen, weights=at, experts=at, order=at, positions=at, offsets=at)
        for name in missing:
            setattr(r, name, None)
        return C.byref(r)
    x, size = matrix(4, 8), C.c_size_t()
    cases = [
        ("expected float, half or bfloat16", lib.qmlp_layer_norm_forward, (matrix(4, 8, _capi.QMLP_DOUBLE), None, None, 1e-5, x, None, None)),
        ("expected half", lib.qmlp_layer_norm_forward, (x, None, None, 1e-5, matrix(4, 8, _capi.QMLP_FLOAT), None, None)),
        ("wrong size at dimension 1", lib.qmlp_layer_norm_forward, (x, None, None, 1e-5, matrix(4, 9), None, None)),
        ("side by side", lib.qmlp_layer_norm_forward, (matrix(4, 8, strides=(1, 4)), None, None, 1e-5, x, None, None)),
        ("overlap", lib.qmlp_layer_norm_forward, (x, None, None, 1e-5, matrix(4, 8, strides=(4, 1)), None, None)),
        ("epsilon", lib.qmlp_layer_norm_forward, (x, None, None, -1.0, x, None, None)),
        ("weight has the wrong data type", lib.qmlp_layer_norm_forward, (x, vector(8, _capi.QMLP_BFLOAT16), None, 1e-5, x, None, None)),
        ("bias must be contiguous", lib.qmlp_layer_norm_forward, (x, None, vector(8, stride=2), 1e-5, x, None, None)),
        ("stats is undefined", lib.qmlp_layer_norm_adjoint, (x, x, None, None, x, None, None, None, None, 0)),
        ("1 to 1048576 channels", lib.qmlp_layer_norm_forward, (matrix(4, 0), None, None, 1e-5, matrix(4, 0), None, None)),
        ("expected int32 or int64", lib.qmlp_embedding_forward, (vector(4), x, 1.0, x, None)),
        ("wrong size at dimension 0", lib.qmlp_embedding_forward, (vector(5, _capi.QMLP_INT64), x, 1.0, x, None)),
        ("impossible size", lib.qmlp_embedding_adjoint_memory, (-1, 4, 8, _capi.QMLP_HALF, C.byref(size))),
        ("1 to 1024 experts", lib.qmlp_route_memory, (routing(experts=1025), C.byref(size))),
        ("a row chooses 1 to 32", lib.qmlp_route_memory, (routing(chosen=9), C.byref(size))),
        ("a row chooses 1 to 32", lib.qmlp_route_memory, (routing(chosen=0), C.byref(size))),
        ("too many rows", lib.qmlp_route_memory, (routing(tokens=2 ** 31), C.byref(size))),
        ("wrong size at dimension 1", lib.qmlp_route_forward, (matrix(4, 9), 1, routing(), None, None, 0)),
        ("order is undefined", lib.qmlp_route_forward, (x, 1, routing(order=None), None, None, 0)),
        ("scratch memory of", lib.qmlp_route_forward, (matrix(40000, 8), 1, routing(tokens=40000), None, None, 0)),
        ("adj_weights is undefined", lib.qmlp_route_adjoint, (x, 1, routing(), None, x, None)),
        ("expected half or bfloat16", lib.qmlp_expert_linear_forward_memory, (matrix(4, 8, _capi.QMLP_FLOAT), matrix(16, 8, _capi.QMLP_FLOAT), 2, C.byref(size))),
        ("1 to 2048 experts", lib.qmlp_expert_linear_forward_memory, (x, matrix(4098, 8), 2049, C.byref(size))),
        ("channels out of 3 experts", lib.qmlp_expert_linear_forward_memory, (x, matrix(16, 8), 3, C.byref(size))),
        ("weight must be contiguous", lib.qmlp_expert_linear_forward_memory, (x, matrix(16, 8, strides=(16, 1)), 2, C.byref(size))),
        ("offsets is undefined", lib.qmlp_expert_linear_forward, (x, matrix(16, 8), None, 2, None, x, None, None, 0)),
        ("bias has the wrong", lib.qmlp_expert_linear_forward, (x, matrix(16, 8), at, 2, vector(16), x, None, None, 0)),
    ]
    for message, function, args in cases:
        assert function(*args) != 0, message
        assert message in lib.qmlp_last_error().decode(), (message, lib.qmlp_last_error())
    # (the networks' own entry points refuse the further types)
    act = C.c_void_p()
    assert lib.qmlp_activation_create(b"relu", C.byref(act)) == 0
    assert lib.qmlp_activation_forward(act, matrix(4, 8, _capi.QMLP_BFLOAT16), matrix(4, 8), None) != 0
    lib.qmlp_activation_destroy(act)
