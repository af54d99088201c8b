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


def test_parameters_of_other_dimensions(qmlp, error):
    """a weight or bias of more dimensions than a view holds, or of none (which is not "no parameter"), or of another width"""
    x, h, r = rand(2, (4, 8)), rand(3, (4, 8), torch.float16), rand(4, (8,))
    y, stats = torch.ops.qmlp_b200.layer_norm_forward(x, r, r, 1e-5)
    for wrong in (r.view(1, 1, 8), r.view(1, 8), r.view(1, 1, 1, 1, 1, 8), r[0], r[:7], torch.tensor(2.0, device="cuda")):
        for weight, bias in ((wrong, None), (None, wrong), (r, wrong)):
            with pytest.raises(error, match="wrong dimension|number of channels"):
                qmlp.layer_norm(x, weight, bias)
            with pytest.raises(error, match="wrong dimension|number of channels"):
                torch.ops.qmlp_b200.layer_norm_adjoint(x, x, weight, bias, stats, True, True, True)
    matrices, offsets = rand(5, (3, 5, 8), torch.float16), torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda")
    b = rand(6, (3, 5), torch.float16)
    for wrong in (b[0, 0], b[0], b[None], b[:, :4], b[:2]):
        with pytest.raises(error):
            qmlp.expert_linear(h, matrices, offsets, wrong)
