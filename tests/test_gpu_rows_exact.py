"""The operators on feature rows where rounding cannot hide a lost term: inputs are small integers, whose sums are exact in 32 bits in
any order, so a result is the exact one, rounded once to its type. Runs that are cut, widths that leave warps and tiles partly empty, any subset of the
gradients."""
import itertools

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu
IDS = {torch.float32: "float", torch.float16: "half", torch.bfloat16: "bfloat16"}


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def whole(seed, shape, dtype, most=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, shape, device="cuda", generator=gen).to(dtype)


def offsets_of(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


def experts_exact(qmlp, counts, n_in, n_out, dtype, wanted=("x", "weight", "bias")):
    rows, experts = sum(counts), len(counts)
    tensors = dict(x=whole(1, (rows, n_in), dtype), weight=whole(2, (experts, n_out, n_in), dtype), bias=whole(3, (experts, n_out), dtype))
    grad, offsets = whole(4, (rows, n_out), dtype), offsets_of(counts)
    exact = dict(zip(("y", "x", "weight", "bias"), (r for r, _ in ref.expert_linear(tensors["x"], tensors["weight"], offsets, tensors["bias"], grad))))
    leaves = {n: t.clone().requires_grad_(n in wanted) for n, t in tensors.items()}
    y = qmlp.expert_linear(leaves["x"], leaves["weight"], offsets, leaves["bias"])
    got = dict(zip(wanted, torch.autograd.grad(y, [leaves[n] for n in wanted], grad)), y=y.detach())
    for name, t in got.items():
        assert exact[name].abs().max() < 2 ** 24 and torch.equal(t, exact[name].to(dtype)), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("counts,n_in,n_out", [([70, 3, 0, 200], 128, 40), ([300], 66, 65), ([9000, 0, 700], 100, 7), ([129, 128, 1], 128, 127),     # both gradients in one pass
                                               ([5000, 20], 200, 72), ([3000, 0, 900], 264, 200), ([20000], 72, 136)])
def test_expert_linear_lanes(qmlp, counts, n_in, n_out, dtype):
    """channels out that leave a warp of the gradients' epilogues with some of its lanes, before and between reads of tensor memory; runs that are cut"""
    experts_exact(qmlp, counts, n_in, n_out, dtype)
