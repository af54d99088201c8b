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
