"""Dropout and the 4-bit operators as far as they go without a GPU: the generator's published answers, the format's packing, shapes, types and gradients on meta
tensors, refusals, tracing, and the argument checks of the C ABI."""
import ctypes as C

import pytest
import torch

import mx_reference as mx


@pytest.fixture(scope="module")
def error():
    import qmlp  # noqa: F401
    from qmlp._capi import QmlpError
    return QmlpError


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("counter,key,words", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_generator(counter, key, words):
    """the known answers that its authors publish with Philox4x32-10"""
    assert tuple(int(w) for w in mx.philox(counter, key)) == words


def test_format():
    """every code's value; ties, borders, saturation; a number is nearest to itself; packing puts every block where it belongs"""
    number = torch.arange(16, dtype=torch.uint8).repeat(2)[None]
    values = mx.values(number, torch.tensor([[128]], dtype=torch.uint8))[0]
    assert values[:8].tolist() == [0, 1, 2, 3, 4, 6, 8, 12] and torch.equal(values[8:16], -values[:8])
    x = torch.tensor([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.26, 0.2, -7.0]])
    assert mx.nearest(x)[0].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -0.5, 0.0, -6.0]
    y = torch.randn(300, 200, generator=torch.Generator().manual_seed(1))
    q = mx.nearest(y)
    again = mx.nearest(torch.where(q.abs() == q.abs().amax(), q, q))
    assert torch.equal(again, q)
    codes, scales = mx.pack(*mx.quantize(y))
    assert codes.shape == (300, 112) and scales.shape == (3, 2, 32, 4, 4)
    for r, c in ((0, 0), (127, 199), (128, 31), (299, 160), (200, 128)):
        code = int(codes[r, c // 2]) >> 4 * (c % 2) & 15
        scale = int(scales[r // 128, c // 128, r % 32, r % 128 // 32, c % 128 // 32])
        assert (-1) ** (code >> 3) * mx.LEVELS[code & 7] * 2.0 ** (scale - 127) == float(q[r, c])


def test_meta():
    """shapes, types and the autograd graph; dropout can be differentiated again, the product cannot"""
    import qmlp
    half = torch.float16
    x, r = meta(6, 10, 24, dtype=half).requires_grad_(), meta(6, 10, 24, dtype=half).requires_grad_()
    y = qmlp.dropout(x, 0.1, 5, residual=r, step=meta(1, dtype=torch.int64))
    grads = torch.autograd.grad(y, [x, r], torch.empty_like(y).requires_grad_(), create_graph=True)
    assert y.shape == x.shape and all(g.shape == x.shape and g.dtype == half for g in grads) and grads[0].requires_grad
    only, = torch.autograd.grad(qmlp.dropout(x.detach(), 0.1, 5, residual=r), [r], torch.empty_like(y))
    assert only.shape == r.shape

    q = qmlp.mx_quantize(meta(3, 130, 77).requires_grad_())
    assert (q.codes.shape, q.scales.shape, q.channels) == ((3, 130, 48), (3, 2, 1, 32, 4, 4), 77) and q.codes.dtype == q.scales.dtype == torch.uint8
    assert not q.codes.requires_grad and qmlp.mx_dequantize(q, torch.bfloat16).shape == (3, 130, 77)
    h, o, b = meta(50, 77, dtype=half).requires_grad_(), meta(4, dtype=torch.int32), meta(3, 130, dtype=half).requires_grad_()
    y = qmlp.mx_linear(h, q, o, b)
    dx, db = torch.autograd.grad(y, [h, b], torch.empty_like(y), create_graph=True)
    assert y.shape == (50, 130) and dx.shape == h.shape and db.shape == b.shape
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    one = qmlp.mx_quantize(meta(40, 77))
    v = meta(40, dtype=half).requires_grad_()
    y = qmlp.mx_linear(meta(2, 5, 77, dtype=half), one, None, v)
    assert y.shape == (2, 5, 40) and torch.autograd.grad(y, v, torch.empty_like(y))[0].shape == (40,)


def test_refusals(error):
    import qmlp
    half = torch.float16
    x, h = meta(10, 40), meta(10, 40, dtype=half)
    q, e, o = qmlp.mx_quantize(meta(24, 40)), qmlp.mx_quantize(meta(3, 24, 40)), meta(4, dtype=torch.int32)
    wrong = [
        ("shape", lambda: qmlp.dropout(x, 0.1, 1, residual=x[:1])), ("type", lambda: qmlp.dropout(x, 0.1, 1, residual=x.half())), ("between", lambda: qmlp.dropout(x, 1.5, 1)),
        ("step", lambda: qmlp.dropout(x, 0.5, 1, step=meta(2, dtype=torch.int64))), ("step", lambda: qmlp.dropout(x, 0.5, 1, step=meta(1))),
        ("channel", lambda: qmlp.dropout(meta(4, 0), 0.1, 1)), ("dimension", lambda: qmlp.dropout(meta(), 0.1, 1)),
        ("needed", lambda: qmlp.mx_quantize(meta(8))), ("needed", lambda: qmlp.mx_quantize(meta(1, 2, 3, 4))), ("channel", lambda: qmlp.mx_quantize(meta(4, 0))),
        ("codes", lambda: qmlp.mx_dequantize(q._replace(channels=65))), ("at least one channel", lambda: qmlp.mx_dequantize(q._replace(channels=0))),
        ("uint8", lambda: qmlp.mx_dequantize(q._replace(codes=meta(24, 32)))), ("scales", lambda: qmlp.mx_dequantize(q._replace(scales=e.scales))),
        ("channels", lambda: qmlp.mx_linear(h[:, :39], q)), ("no offsets", lambda: qmlp.mx_linear(h, q, o)), ("need offsets", lambda: qmlp.mx_linear(h, e)),
        ("bias", lambda: qmlp.mx_linear(h, q, None, meta(1, 24, dtype=half))), ("bias", lambda: qmlp.mx_linear(h, q, None, meta(23, dtype=half))),
        ("bias", lambda: qmlp.mx_linear(h, e, o, meta(24, dtype=half))), ("row per expert", lambda: qmlp.mx_linear(h, e, o, meta(2, 24, dtype=half))),
    ]
    for message, call in wrong:
        with pytest.raises(error, match=message):
            call()
            print("not refused:", message)
    ones = torch.ones((4, 32))
    cpu = qmlp.MXTensor(torch.zeros((8, 16), dtype=torch.uint8), torch.zeros((1, 1, 32, 4, 4), dtype=torch.uint8), 32)
    for call in (lambda: qmlp.dropout(ones, 0.1, 1), lambda: qmlp.mx_quantize(ones), lambda: qmlp.mx_dequantize(cpu), lambda: qmlp.mx_linear(ones.half(), cpu)):
        with pytest.raises(error, match="CUDA"):
            call()
    for bad in (-0.1, 1.1):
        with pytest.raises(ValueError):
            qmlp.FusedDropout(bad, device="meta")


def test_forward_mode(error):
    """no tangent is dropped in silence"""
    import torch.autograd.forward_ad as fwad
    import qmlp
    q, o = qmlp.mx_quantize(meta(3, 24, 40)), meta(4, dtype=torch.int32)
    calls = [(lambda x, r: qmlp.dropout(x, 0.1, 1, residual=r), [meta(4, 8), meta(4, 8)]),
             (lambda x, b: qmlp.mx_linear(x, q, o, b), [meta(6, 40, dtype=torch.float16), meta(3, 24, dtype=torch.float16)]),
             (lambda g: torch.ops.qmlp_b200.mx_linear_adjoint(g, q.codes, q.scales, 40, o, True, False)[0], [meta(6, 24, dtype=torch.float16)])]
    for call, args in calls:
        for i, a in enumerate(args):
            with fwad.dual_level(), pytest.raises(error, match="forward-mode"):
                call(*args[:i], fwad.make_dual(a, torch.empty_like(a)), *args[i + 1:])


def test_traceable():
    """torch.compile takes the functions and the modules whole"""
    import qmlp
    half = torch.float16
    seen = []

    def backend(graph, inputs):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    def model(x, r, w, b):
        q = qmlp.mx_quantize(w)
        return qmlp.mx_linear(qmlp.dropout(x, 0.1, 3, residual=r), q, None, b) + qmlp.mx_dequantize(q, half).sum()
    args = [meta(30, 40, dtype=half).requires_grad_(), meta(30, 40, dtype=half), meta(16, 40), meta(16, dtype=half)]
    torch._dynamo.reset()
    y = torch.compile(model, fullgraph=True, backend=backend)(*args)
    assert y.shape == (30, 16) and all(any(name in t for t in seen) for name in ("dropout_forward", "mx_quantize", "mx_linear_forward", "mx_dequantize")), seen
    y = torch.compile(model, fullgraph=True, backend="aot_eager")(*args)
    assert torch.autograd.grad(y, args[0], torch.empty_like(y))[0].shape == (30, 40)
    layer = qmlp.FusedExperts(16, 32, 8, experts=4, dtype=torch.bfloat16, device="meta", dropout=0.2)
    assert torch.compile(layer, fullgraph=True, backend="aot_eager")(meta(5, 3, 16)).shape == (5, 3, 8)
    assert torch.compile(layer.quantized().eval(), fullgraph=True, backend="aot_eager")(meta(5, 3, 16)).shape == (5, 3, 8)
    torch._dynamo.reset()


def test_modules():
    """what a layer without dropout holds is as it was; parameters and buffers of the others"""
    import qmlp
    plain, dropping = (qmlp.FusedExperts(16, 32, 8, experts=4, dtype=torch.bfloat16, device="meta", dropout=p) for p in (0.0, 0.3))
    assert list(plain.state_dict()) == ["router", "weight1", "bias1", "weight2", "bias2"] and plain.dropout is None
    assert "dropout.step" in dropping.state_dict() and dropping.dropout.p == 0.3
    served = plain.quantized()
    assert not list(served.parameters()) and served.codes1.shape == (4, 32, 16) and served.codes2.shape == (4, 8, 16) and served(meta(7, 16)).shape == (7, 8)


def test_c_abi_refusals():
    """checks that come before anything touches a device; the pointers are never followed"""
    from qmlp import _capi
    lib = _capi.lib()
    here = C.create_string_buffer(4096)
    at = (C.addressof(here) + 255) // 256 * 256

    def matrix(rows, channels, precision=_capi.QMLP_HALF, strides=None, data=at):
        t = _capi.Tensor(data=data, precision=precision, ndim=2)
        t.sizes[0], t.sizes[1] = rows, channels
        t.strides[0], t.strides[1] = strides or (channels, 1)
        return C.byref(t)

    def mxm(matrices=1, rows=8, channels=8, codes=at, scales=at):
        return C.byref(_capi.Mx(matrices=matrices, rows=rows, channels=channels, codes=codes, scales=scales))
    x, size, other = matrix(4, 8), C.c_size_t(), C.c_size_t()
    assert lib.qmlp_mx_memory(3, 130, 77, C.byref(size), C.byref(other)) == 0 and (size.value, other.value) == (3 * 130 * 48, 3 * 2 * 512)
    cases = [
        ("expected float, half or bfloat16", lib.qmlp_dropout, (matrix(4, 8, _capi.QMLP_DOUBLE), None, 0.1, 1, 0, None, x, None)),
        ("output has the wrong data type", lib.qmlp_dropout, (x, None, 0.1, 1, 0, None, matrix(4, 8, _capi.QMLP_FLOAT), None)),
        ("wrong size at dimension 0", lib.qmlp_dropout, (x, matrix(5, 8), 0.1, 1, 0, None, x, None)),
        ("overlap", lib.qmlp_dropout, (x, None, 0.1, 1, 0, None, matrix(4, 8, strides=(4, 1)), None)),
        ("probability", lib.qmlp_dropout, (x, None, -0.1, 1, 0, None, x, None)),
        ("probability", lib.qmlp_dropout, (x, None, float("nan"), 1, 0, None, x, None)),
        ("channels", lib.qmlp_mx_memory, (1, 8, 0, C.byref(size), C.byref(other))),
        ("too many rows", lib.qmlp_mx_memory, (1 << 20, 1 << 20, 8, C.byref(size), C.byref(other))),
        ("too many tiles", lib.qmlp_mx_memory, (1, 1 << 30, 1 << 20, C.byref(size), C.byref(other))),
        ("code_bytes is undefined", lib.qmlp_mx_memory, (1, 8, 8, None, C.byref(other))),
        ("output is undefined", lib.qmlp_mx_quantize, (x, None, None)),
        ("output is undefined", lib.qmlp_mx_quantize, (matrix(8, 8), mxm(codes=None), None)),
        ("16-byte aligned", lib.qmlp_mx_quantize, (matrix(8, 8), mxm(scales=at + 8), None)),
        ("wrong size at dimension 0", lib.qmlp_mx_quantize, (x, mxm(), None)),
        ("wrong size at dimension 1", lib.qmlp_mx_dequantize, (mxm(), matrix(8, 9), None)),
        ("weight is undefined", lib.qmlp_mx_linear_forward_memory, (x, None, C.byref(size))),
        ("expected half or bfloat16", lib.qmlp_mx_linear_forward_memory, (matrix(4, 8, _capi.QMLP_FLOAT), mxm(), C.byref(size))),
        ("1 to 2048 experts", lib.qmlp_mx_linear_forward_memory, (x, mxm(matrices=2049), C.byref(size))),
        ("1 to 2048 experts", lib.qmlp_mx_linear_forward_memory, (x, mxm(matrices=0), C.byref(size))),
        ("channels out", lib.qmlp_mx_linear_forward_memory, (x, mxm(rows=0), C.byref(size))),
        ("wrong size at dimension 1", lib.qmlp_mx_linear_forward_memory, (x, mxm(channels=9), C.byref(size))),
        ("too many rows", lib.qmlp_mx_linear_forward_memory, (matrix((1 << 31) - 8192, 1 << 20), mxm(channels=1 << 20), C.byref(size))),
        ("offsets is undefined", lib.qmlp_mx_linear_forward, (x, mxm(matrices=2), None, None, x, None, None, 0)),
        ("output has the wrong size", lib.qmlp_mx_linear_forward, (x, mxm(), None, None, matrix(4, 9), None, None, 0)),
        ("bias has the wrong", lib.qmlp_mx_linear_forward, (x, mxm(), None, matrix(2, 8), x, None, None, 0)),
        ("adj_input has the wrong", lib.qmlp_mx_linear_adjoint, (x, mxm(), None, matrix(4, 9), None, None, None, 0)),
    ]
    for message, function, args in cases:
        assert function(*args) != 0, message
        assert message in lib.qmlp_last_error().decode(), (message, lib.qmlp_last_error())
