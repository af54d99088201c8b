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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("experts", [60, 700])
def test_expert_linear_slots(qmlp, experts, dtype):
    """cut runs between whole and empty ones, in order of length (up to 512 experts) and not: each finds the partial sums that are its own"""
    counts = [0] * experts
    for i, n in enumerate((3, 1700, 0, 1, 2100, 5, 40, 0, 5000, 512, 513, 511, 2100, 64, 1025)):
        counts[i * 4 + i % 3] = n
    counts[-1] = 3000
    experts_exact(qmlp, counts, 200, 136, dtype)
    experts_exact(qmlp, counts, 136, 40, dtype, ("weight",))


def test_expert_linear_scratch(qmlp):
    """the scratch of a weight gradient follows the runs that can be cut: no copy of all matrices"""
    import ctypes as C
    from qmlp import _capi
    lib = _capi.lib()

    def matrix(rows, channels):
        t = _capi.Tensor(data=1 << 20, precision=_capi.QMLP_HALF, ndim=2)     # (the pointers are not followed)
        t.sizes[0], t.sizes[1], t.strides[0], t.strides[1] = rows, channels, channels, 1
        return C.byref(t)

    for rows, experts, n_in, n_out in ((131072, 512, 1024, 1024), (131072, 256, 2048, 2048), (600, 256, 1024, 4096), (131072, 512, 1024, 4096), (1 << 20, 2048, 512, 512),
                                       (2000, 2048, 1024, 1024)):
        size = C.c_size_t()
        assert lib.qmlp_expert_linear_adjoint_memory(matrix(rows, n_in), matrix(rows, n_out), matrix(experts * n_out, n_in), experts, _capi.GRADIENTS_INPUT | _capi.GRADIENTS_NETWORK_WEIGHTS,
                                                     C.byref(size)) == 0
        assert size.value < 2 * experts * n_in * n_out / 4, (experts, size.value)
