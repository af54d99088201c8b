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


WANTED = [w for n in (1, 2, 3) for w in itertools.combinations(("x", "weight", "bias"), n)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("wanted", WANTED, ids="+".join)
def test_expert_linear_wanted(qmlp, wanted, dtype):
    """any subset of the gradients: layers on both sides of 128 channels (one pass for two gradients, or a kernel each), odd widths that are copied
    first, cut and empty runs, few rows, one expert"""
    for counts, n_in, n_out in (([300, 0, 45, 1100], 64, 64), ([3000, 0, 40], 128, 128), ([700, 2, 0, 1900], 136, 200), ([600, 30], 31, 130), ([513, 0, 5000], 520, 264),
                                ([5, 0, 1], 77, 40), ([1], 8, 8), ([4000], 13, 129), ([0, 0, 200], 256, 64)):
        experts_exact(qmlp, counts, n_in, n_out, dtype, wanted)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("wanted", WANTED, ids="+".join)
@pytest.mark.parametrize("rows,channels", [(40003, 48), (3001, 64), (2500, 37), (3001, 512), (1500, 1024), (700, 777), (900, 2048), (401, 4096), (300, 8192), (160, 16384), (150, 16392)])
def test_layer_norm_wanted(qmlp, rows, channels, wanted, dtype):
    """any subset of the gradients, from whole means and a deviation of one: sums over rows are exact, and over channels where they are a power of two"""
    x, grad, weight = whole(11, (rows, channels), dtype, 3), whole(12, (rows, channels), dtype), whole(13, (channels,), torch.float32)
    mean = whole(14, (rows,), torch.float32, 1)
    stats = torch.stack([mean, torch.ones_like(mean)])
    got = torch.ops.qmlp_b200.layer_norm_adjoint(x, grad, weight, weight, stats, *(n in wanted for n in ("x", "weight", "bias")))
    u, g = x.double() - mean[:, None].double(), grad.double()
    gw = g * weight.double()
    exact = [gw - gw.mean(1, keepdim=True) - u * (gw * u).mean(1, keepdim=True), (g * u).sum(0), g.sum(0)]
    for name, t, e in zip(("x", "weight", "bias"), got, exact):
        if name not in wanted:
            assert t.numel() == 0
        elif name != "x":
            assert t.dtype == torch.float32 and torch.equal(t.double(), e), name
        elif channels & (channels - 1) == 0:
            assert e.abs().max() < 2 ** 10 and torch.equal(t, e.to(dtype)), name      # (multiples of 1 / channels below 1024: 24 bits)
        else:
            size = gw.abs() + gw.abs().mean(1, keepdim=True) + u.abs() * (gw * u).abs().mean(1, keepdim=True)
            ref.check(t, e, ref.sum_slack(channels, size), name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("tokens,rows,channels", [(310001, 700, 8), (60000, 3, 33), (40000, 1, 64), (30000, 20000, 40), (4097, 50, 1030), (100003, 1500, 16)])
def test_embedding_exact(qmlp, tokens, rows, channels, dtype):
    """the table's gradient to the last term: short and long runs, runs that cross many chunks"""
    gen = torch.Generator(device="cuda").manual_seed(21)
    at = torch.randint(-1, rows + 1, (tokens,), device="cuda", generator=gen)
    at = torch.where(torch.rand(tokens, device="cuda", generator=gen) < 0.3, rows // 2, at)
    grad = whole(22, (tokens, channels), dtype)
    table = whole(23, (rows, channels), dtype).requires_grad_()
    got, = torch.autograd.grad(qmlp.embedding(at, table, 2.0), table, grad)
    inside = (at >= 0) & (at < rows)
    exact = torch.zeros((rows, channels), dtype=torch.float64, device="cuda").index_add_(0, at[inside], grad[inside].double()) * 2
    assert torch.equal(got, exact.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("rows,experts,k,channels", [(3000, 9, 1, 64), (3000, 9, 2, 264), (2000, 40, 3, 37), (1500, 8, 8, 50), (700, 33, 32, 8), (60, 4, 2, 4104)])
def test_exchange_exact(qmlp, rows, experts, k, channels, dtype):
    """both directions of the movement of rows and all gradients to the last term, with slots that have no expert"""
    gen = torch.Generator(device="cuda").manual_seed(31)
    z = torch.randn((rows, experts), device="cuda", generator=gen)
    z[torch.rand((rows, experts), device="cuda", generator=gen) < 0.4] = -float("inf")
    z[0] = -float("inf")
    r = qmlp.route(z, k)
    w = whole(32, (rows, k), torch.float32).requires_grad_()
    x, y = whole(33, (rows, channels), dtype).requires_grad_(), whole(34, (rows * k, channels), dtype).requires_grad_()
    gx, gy = whole(35, (rows * k, channels), dtype), whole(36, (rows, channels), dtype)
    sent, back = qmlp.dispatch(x, r), qmlp.combine(y, r._replace(weights=w))
    dx, dy, dw = torch.autograd.grad([sent, back], [x, y, w], [gx, gy])
    have, at, used = (r.positions >= 0)[:, :, None], r.positions.clamp(min=0).long(), (r.order >= 0)[:, None]
    token, y64, g64 = r.order.clamp(min=0).long() // k, y.detach().double()[at] * have, gy.double()
    slot_w = w.detach().reshape(-1)[r.order.clamp(min=0).long()][:, None].double()
    for name, got, exact in (("dispatch", sent.detach(), x.detach().double()[token] * used), ("combine", back.detach(), (w.detach().double()[:, :, None] * y64).sum(1)),
                             ("input gradient", dx, (gx.double()[at] * have).sum(1)), ("rows' gradient", dy, slot_w * g64[token] * used),
                             ("weights' gradient", dw, (y64 * g64[:, None]).sum(2))):
        assert torch.equal(got, exact.to(got.dtype)), name
