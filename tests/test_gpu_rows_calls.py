"""Calls of the operators on feature rows that are refused, or that ask for less than everything: what comes back is right or an error."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


@pytest.fixture(scope="module")
def error(qmlp):
    from qmlp._capi import QmlpError
    return QmlpError


def rand(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(dtype)


def test_layer_norm_stats(qmlp, error):
    """the adjoint reads a mean and a deviation per row: statistics of another size, type or layout are refused"""
    x = rand(1, (30, 8))
    y, stats = torch.ops.qmlp_b200.layer_norm_forward(x, None, None, 1e-5)
    assert torch.ops.qmlp_b200.layer_norm_adjoint(x, x, None, None, stats, True, False, False)[0].shape == x.shape
    for wrong in (stats[:, 1:], stats[:, :29].contiguous(), stats.reshape(-1), stats.half(), stats.t().contiguous().t(), stats[:, :0]):
        with pytest.raises(error, match="stats"):
            torch.ops.qmlp_b200.layer_norm_adjoint(x, x, None, None, wrong, True, False, False)
