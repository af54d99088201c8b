"""4-bit matrices as far as it goes without a GPU: what autograd is told of them, layers that are cast as a whole."""
import pytest
import torch


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_quantize_refuses_tangents(qmlp):
    """no tangent is dropped in silence: not by the function, not by the operator; codes cannot have one"""
    import torch.autograd.forward_ad as fwad
    from qmlp._capi import QmlpError
    for call in (qmlp.mx_quantize, torch.ops.qmlp_b200.mx_quantize):
        call(meta(8, 40))
        with fwad.dual_level(), pytest.raises(QmlpError, match="forward-mode"):
            call(fwad.make_dual(meta(8, 40), meta(8, 40)))
    codes = qmlp.mx_quantize(meta(8, 40)).codes
    with fwad.dual_level(), pytest.raises(ValueError, match="floating"):
        fwad.make_dual(codes, codes)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_served_layers_are_cast(qmlp, dtype, monkeypatch):
    """a model with a served layer that is cast as a whole still runs: what the products are given has their type (meta tensors do not see to that)"""
    linear, mx_linear = torch.nn.functional.linear, qmlp.rows.mx_linear

    def checked_linear(x, w):
        assert x.dtype == w.dtype == torch.float32
        return linear(x, w)

    def checked_mx_linear(x, weight, offsets, bias):
        assert x.dtype == bias.dtype == dtype
        return mx_linear(x, weight, offsets, bias)
    monkeypatch.setattr(torch.nn.functional, "linear", checked_linear)
    monkeypatch.setattr(qmlp.rows, "mx_linear", checked_mx_linear)
    for cast in (torch.float16, torch.bfloat16, torch.float32, torch.float64):
        served = qmlp.FusedExperts(16, 32, 8, experts=4, dtype=dtype, device="meta").quantized().to(cast)
        y = served(meta(7, 16, dtype=cast))
        assert served.bias1.dtype == cast and served.codes1.dtype == torch.uint8 and y.shape == (7, 8) and y.dtype == dtype


def test_layers_in_64_bits_are_served(qmlp, monkeypatch):
    """parameters in float64, which a layer casts per call, are rounded to float32 first (meta tensors would take any type)"""
    seen = []
    quantize = qmlp.rows.mx_quantize
    monkeypatch.setattr(qmlp.rows, "mx_quantize", lambda w: seen.append(w.dtype) or quantize(w))
    for given, taken in ((torch.float64, torch.float32), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)):
        layer = qmlp.FusedExperts(16, 32, 8, experts=4, weight_dtype=given, device="meta")
        served = layer.quantized()
        assert seen == [taken] * 2 and served(meta(7, 16)).shape == layer(meta(7, 16)).shape
        seen.clear()
