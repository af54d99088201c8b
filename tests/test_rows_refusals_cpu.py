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
