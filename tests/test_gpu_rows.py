"""The operators on feature rows (layer norm, embedding lookup, routing, products grouped by expert) against their definitions
in 64 bits (rows_reference.py): types, odd sizes, strides, empty and masked rows, gradients, streams, refusals."""
import json

import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu
FLOATS = [torch.float32, torch.float16, torch.bfloat16]
IDS = {torch.float32: "float", torch.float16: "half", torch.bfloat16: "bfloat16"}
INF = float("inf")


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(dtype)


def ints(seed, shape, low, high, dtype=torch.int64):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, shape, device="cuda", generator=gen, dtype=dtype)


# ---- layer norm --------------------------------------------------------------------------------------------------------
def layer_norm_case(qmlp, x, weight, bias, grad, eps=1e-5):
    x = x.detach().requires_grad_()
    params = [p.detach().requires_grad_() if p is not None else None for p in (weight, bias)]
    y = qmlp.layer_norm(x, params[0], params[1], eps)
    got = torch.autograd.grad(y, [x] + [p for p in params if p is not None], grad)
    exact = ref.layer_norm(x.detach(), weight, bias, eps, grad)
    assert y.dtype == x.dtype and y.shape == x.shape
    ref.check(y.detach(), *exact[0], "output")
    ref.check(got[0], *exact[1], "input gradient")
    at = 1
    for p, e, name in ((weight, exact[2], "weight gradient"), (bias, exact[3], "bias gradient")):
        if p is not None:
            assert got[at].dtype == p.dtype
            ref.check(got[at], *e, name)
            at += 1


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("rows,channels", [(1, 512), (3, 1), (1000, 8), (517, 13), (65, 64), (33, 65), (700, 200), (130, 256), (19, 264), (77, 512), (5, 777),
                                           (40, 1024), (9, 1032), (300, 2048), (7, 2049), (11, 4096), (6, 5000), (3, 8192), (2, 9001), (4, 16384), (3, 16385), (2, 20001)])
def test_layer_norm(qmlp, rows, channels, dtype):
    x, grad = rand(1, (rows, channels), dtype, 1.5, 0.3), rand(2, (rows, channels), dtype)
    layer_norm_case(qmlp, x, rand(3, (channels,), std=0.2, mean=1.0), rand(4, (channels,), std=0.2), grad)


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
def test_layer_norm_parameters(qmlp, dtype):
    """without parameters, with one of them, with parameters of the features' type; a large batch over many blocks"""
    x, grad = rand(5, (40003, 48), dtype), rand(6, (40003, 48), dtype)
    w, b = rand(7, (48,), mean=1.0), rand(8, (48,))
    for weight, bias in ((None, None), (w, None), (None, b), (w.to(dtype), b.to(dtype)), (w, b)):
        layer_norm_case(qmlp, x, weight, bias, grad)


def test_layer_norm_strides(qmlp):
    """rows apart, rows that start off a 16-byte boundary, transposed and expanded tensors, more than two dimensions"""
    base = rand(9, (300, 130), torch.float16)
    w, b = rand(10, (96,), mean=1.0), rand(11, (96,))
    for x in (base[:, :96], base[:, 1:97], base[::3, 8:104], rand(12, (96, 50), torch.float16).t(), rand(13, (1, 96), torch.float16).expand(20, 96)):
        layer_norm_case(qmlp, x, w, b, rand(14, tuple(x.shape), torch.float16))
        layer_norm_case(qmlp, x.contiguous(), w, b, rand(15, (1, 96), torch.float16).expand(x.shape))
    x = rand(16, (4, 7, 96))
    y = qmlp.layer_norm(x, w, b)
    assert y.shape == x.shape and torch.equal(y.reshape(28, 96), qmlp.layer_norm(x.reshape(28, 96), w, b))


def test_layer_norm_values(qmlp):
    """constant rows (no variance), a large common offset, large values; NaN and infinity stay in their row"""
    x = rand(17, (64, 100))
    x[0], x[1] = 0.0, 3.0
    x[2] += 1000.0
    x[3] *= 1e15
    layer_norm_case(qmlp, x, rand(18, (100,)), rand(19, (100,)), rand(20, (64, 100)))
    x[5, 3], x[6, 4] = float("nan"), INF
    y = qmlp.layer_norm(x)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[5] = bad[6] = True
    assert torch.equal(torch.isnan(y).any(1), bad)


def test_layer_norm_empty(qmlp):
    x, w = torch.empty((0, 32), device="cuda", requires_grad=True), torch.ones(32, device="cuda", requires_grad=True)
    y = qmlp.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.empty((0, 32), device="cuda"))
    assert y.shape == (0, 32) and dx.shape == (0, 32) and torch.equal(dw, torch.zeros(32, device="cuda"))


def test_layer_norm_differences(qmlp):
    """the gradient along a direction against a central difference: off by the third derivative's share of h^2, and by 2^-22 of the
    output's magnitude over h"""
    x, w, b, g = rand(21, (8, 40)), rand(22, (40,), mean=1.0), rand(23, (40,)), rand(24, (8, 40))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(qmlp.layer_norm(*leaves), leaves, g)
    h = 2.0 ** -7
    for i, t in enumerate((x, w, b)):
        d = rand(25 + i, tuple(t.shape))
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = t + h * d, t - h * d
        up, down = ((qmlp.layer_norm(*a).double() * g).sum() for a in args)
        size = (g.abs() * qmlp.layer_norm(x, w, b).abs()).sum().item()
        assert abs((up - down).item() / (2 * h) - (grads[i].double() * d).sum().item()) < size * (60 * h * h + 2.0 ** -22 / h)


# ---- embedding -----------------------------------------------------------------------------------------------------------
def embedding_case(qmlp, tokens, table, scale, grad):
    leaf = table.detach().requires_grad_()
    y = qmlp.embedding(tokens, leaf, scale)
    dt, = torch.autograd.grad(y, [leaf], grad)
    exact = ref.embedding(tokens, table, scale, grad)
    assert y.shape == (*tokens.shape, table.shape[1]) and y.dtype == table.dtype and dt.dtype == table.dtype
    ref.check(y.detach(), *exact[0], "output")
    ref.check(dt, *exact[1], "table gradient")
    again, = torch.autograd.grad(qmlp.embedding(tokens, leaf, scale), [leaf], grad)
    assert torch.equal(again, dt)      # the same every run


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("tokens,rows,channels", [(1, 1, 1), (1, 1000, 64), (7, 3, 8), (100, 1, 33), (2048, 17, 32), (2049, 1023, 4), (5000, 1024, 16),
                                                  (3001, 1025, 100), (70000, 300, 24), (20000, 40000, 7), (300, 100000, 256), (4097, 50, 1030), (310001, 700, 8), (320000, 3000, 5)])
def test_embedding(qmlp, tokens, rows, channels, dtype):
    t = ints(30, (tokens,), -2, rows + 2)       # a few outside the table
    embedding_case(qmlp, t, rand(31, (rows, channels), dtype), 1.0 if channels % 2 else channels ** 0.5, rand(32, (tokens, channels), dtype))


@pytest.mark.parametrize("kind", ["hot", "one", "masked", "last"])
def test_embedding_runs(qmlp, kind):
    """runs of a token that cross many chunks, tokens that are all the same, all masked, all the last row"""
    n, rows = 30011, 5000
    t = ints(33, (n,), 0, rows)
    if kind == "hot":
        t = torch.where(ints(34, (n,), 0, 3) > 0, 7, t)
    else:
        t[:] = {"one": 0, "masked": -1, "last": rows - 1}[kind]
    embedding_case(qmlp, t, rand(35, (rows, 40)), 1.0, rand(36, (n, 40)))


def test_embedding_layouts(qmlp):
    """int32 tokens, strided tokens, several dimensions, a table and gradients with rows apart or off a 16-byte boundary"""
    table = rand(37, (90, 70), torch.float16)
    tokens = ints(38, (60, 4), -1, 90)
    grad = rand(39, (60, 4, 64), torch.float16)
    embedding_case(qmlp, tokens, table[:, :64], 1.0, grad)
    embedding_case(qmlp, tokens.int(), table[:, 3:67], 2.0, grad)
    embedding_case(qmlp, tokens[:, 1], table[::2, :64], 0.5, rand(40, (60, 70), torch.float16)[:, 2:66])
    embedding_case(qmlp, tokens, table[:, :64], 1.0, rand(41, (1, 1, 64), torch.float16).expand(60, 4, 64))
    embedding_case(qmlp, tokens[:0], table, 1.0, rand(42, (0, 4, 70), torch.float16))
    huge = torch.tensor([2 ** 40, -2 ** 40, 5, 2 ** 31, 2 ** 32 + 5], device="cuda")
    embedding_case(qmlp, huge, table, 1.0, rand(43, (5, 70), torch.float16))


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("channels", [2, 50, 49])
def test_embedding_narrow_rows(qmlp, channels, dtype):
    """rows that allow accesses of two elements or one; tables whose tokens are sorted in one pass and in two"""
    for tokens, rows in ((3000, 700), (6000, 2000), (300, 40000)):
        t = ints(48, (tokens,), -2, rows + 2)
        embedding_case(qmlp, t, rand(49, (rows, channels), dtype), 0.5, rand(53, (tokens, channels), dtype))
    wider = rand(54, (700, channels + 3), dtype)
    for first in (1, 2):
        embedding_case(qmlp, ints(55, (500,), 0, 700), wider[:, first:first + channels], 1.0, rand(56, (500, channels), dtype))


def test_embedding_difference(qmlp):
    """linear in the table: the difference of two outputs is the output of the difference, and pairs with the gradient"""
    tokens, table, d, g = ints(44, (500,), 0, 40), rand(45, (40, 12)), rand(46, (40, 12)), rand(47, (500, 12))
    leaf = table.clone().requires_grad_()
    dt, = torch.autograd.grad(qmlp.embedding(tokens, leaf, 3.0), [leaf], g)
    moved = ((qmlp.embedding(tokens, table + d, 3.0).double() - qmlp.embedding(tokens, table - d, 3.0)) / 2 * g).sum().item()
    size = (qmlp.embedding(tokens, table.abs() + d.abs(), 3.0) * g.abs()).sum().item()
    assert abs(moved - (dt.double() * d).sum().item()) < 520 * 2.0 ** -22 * size


# ---- routing -----------------------------------------------------------------------------------------------------------
def route_case(qmlp, logits, k, normalize):
    leaf = logits.detach().requires_grad_()
    r = qmlp.route(leaf, k, normalize)
    weights, experts, order, positions, offsets = ref.route(logits, k, normalize)
    for got, want, name in ((r.experts, experts, "experts"), (r.order, order, "order"), (r.positions, positions, "positions"), (r.offsets, offsets, "offsets")):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), name
    ref.check(r.weights.detach(), weights.cuda(), ref.sum_slack(logits.shape[1] + 16, weights.cuda()), "weights")
    grad = rand(50, tuple(r.weights.shape))
    dz, = torch.autograd.grad(r.weights, [leaf], grad)
    assert dz.dtype == logits.dtype
    ref.check(dz, *ref.route_gradient(logits, r.experts, weights, grad, normalize), "logits' gradient")


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (1, 64, 2), (3, 8, 8), (513, 5, 2), (600, 16, 3), (1025, 30, 1), (257, 64, 8), (2000, 100, 2), (100, 256, 32),
                                            (90, 257, 4), (70, 1024, 32), (1500, 64, 2)])
def test_route(qmlp, rows, experts, k, normalize, dtype):
    z = rand(51, (rows, experts), dtype, 1.5)
    z[ints(52, (rows, experts), 0, 8) == 0] = -INF
    if rows > 3:
        z[1] = -INF                             # a row whose mask leaves nothing
        z[2] = torch.finfo(dtype).min           # a mask of the type's lowest value: all the same, the first k
        z[3, : experts // 2] = z[3, 0]
    route_case(qmlp, z, k, normalize)


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("rows,experts,k", [(20000, 64, 2), (16385, 8, 1), (17001, 256, 8), (16384, 40, 3), (16500, 136, 5), (66000, 64, 2), (65536, 256, 8), (65601, 40, 1),
                                            (16400, 32, 2), (3000, 64, 2)])
def test_route_many_rows(qmlp, rows, experts, k, normalize, dtype):
    """the kernels for many rows choose and weigh as those for few do, row by row, and order the slots as a sort does"""
    z = rand(59, (rows, experts), dtype, 1.5)
    z[ints(60, (rows, experts), 0, 8) == 0] = -INF
    z[1], z[2], z[3, : experts // 2], z[4, 0], z[5, 1] = -INF, torch.finfo(dtype).min, z[3, 0], float("nan"), INF
    leaf = z.clone().requires_grad_()
    r = qmlp.route(leaf, k, normalize)
    grad = rand(61, (rows, k))
    dz, = torch.autograd.grad(r.weights, [leaf], grad)
    for first in range(0, rows, 7000):
        part = z[first:first + 7000].clone().requires_grad_()
        few = qmlp.route(part, k, normalize)
        rows_of = slice(first, first + 7000)
        assert torch.equal(r.experts[rows_of], few.experts)
        assert torch.allclose(r.weights[rows_of].detach(), few.weights.detach(), rtol=(experts + 16) * 2.0 ** -22, atol=0, equal_nan=True)
        d, = torch.autograd.grad(few.weights, [part], grad[rows_of])
        fine = torch.isfinite(few.weights).all(1)
        w, s = ref.route_gradient(part.detach()[fine], few.experts[fine], few.weights.detach()[fine], grad[rows_of][fine], normalize)
        ref.check(dz[rows_of][fine], w, s, "logits' gradient")
        assert torch.equal(torch.isnan(dz[rows_of]), torch.isnan(d))
    flat = torch.where(r.experts < 0, experts, r.experts).reshape(-1)
    order = torch.argsort(flat, stable=True).int()
    used = int((flat < experts).sum())
    assert torch.equal(r.order[:used], order[:used]) and (r.order[used:] == -1).all()
    assert torch.equal(r.offsets, torch.nn.functional.pad(torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0), (1, 0)).int())


def test_route_values(qmlp):
    """equal zeros of both signs, infinity, NaN: the largest first, NaN before all, weights as a softmax says"""
    z = rand(53, (6, 12))
    z[0] = torch.tensor([0.0, -0.0] * 6, device="cuda")
    z[1, 5] = INF
    z[2, 7] = float("nan")
    z[2, 9] = float("nan")
    r = qmlp.route(z, 3)
    weights, experts, order, positions, offsets = ref.route(z, 3, True)
    assert torch.equal(r.experts.cpu(), experts) and torch.equal(r.order.cpu(), order)
    assert torch.isnan(r.weights[1:3]).all() and torch.isfinite(r.weights[[0, 3, 4, 5]]).all()
    assert r.experts[2, 0] == 7 and r.experts[2, 1] == 9


def test_route_layouts(qmlp):
    base = rand(54, (700, 80), torch.float16)
    for z in (base[:, :64], base[:, 3:67], base[::2, :64], rand(55, (64, 90), torch.float16).t()):
        route_case(qmlp, z, 2, True)
    r = qmlp.route(torch.empty((0, 16), device="cuda"), 2)
    assert r.order.numel() == 0 and torch.equal(r.offsets, torch.zeros(17, dtype=torch.int32, device="cuda"))


def test_route_difference(qmlp):
    """the gradient along a direction that keeps the choice, against a central difference"""
    for normalize in (True, False):
        z, d = rand(56, (50, 20), std=2.0), rand(57, (50, 20))
        leaf = z.clone().requires_grad_()
        r = qmlp.route(leaf, 4, normalize)
        g = rand(58, (50, 4))
        dz, = torch.autograd.grad(r.weights, [leaf], g)
        h = 2.0 ** -10
        up, down = qmlp.route(z + h * d, 4, normalize), qmlp.route(z - h * d, 4, normalize)
        same = (up.experts == r.experts).all(1) & (down.experts == r.experts).all(1)
        assert same.sum() > 40
        moved = ((up.weights.double() - down.weights) * g)[same].sum().item() / (2 * h)
        size = g.abs().sum().item()
        assert abs(moved - (dz.double() * d)[same].sum().item()) < size * (60 * h * h + 2.0 ** -22 / h)


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("rows,experts,k,channels", [(1, 4, 2, 8), (100, 3, 1, 1), (333, 8, 3, 17), (257, 64, 2, 256), (50, 16, 5, 1000), (40, 8, 8, 2049),
                                                     (120, 5, 2, 50), (90, 4, 1, 6), (70, 9, 3, 270)])
def test_exchange(qmlp, rows, experts, k, channels, dtype):
    z = rand(60, (rows, experts))
    z[ints(61, (rows, experts), 0, 3) == 0] = -INF       # slots without an expert
    r = qmlp.route(z, k)
    w = r.weights.clone().requires_grad_()
    r = r._replace(weights=w)
    x, y = rand(62, (rows, channels), dtype).requires_grad_(), rand(63, (rows * k, channels), dtype).requires_grad_()
    sent, back = qmlp.dispatch(x, r), qmlp.combine(y, r)
    g1, g2 = rand(64, (rows * k, channels), dtype), rand(65, (rows, channels), dtype)
    dx, dy, dw = torch.autograd.grad([sent, back], [x, y, w], [g1, g2])
    used = r.order >= 0
    slot = torch.where(used, r.order, 0).long()
    assert torch.equal(sent.detach(), torch.where(used[:, None], x.detach()[slot // k], torch.zeros((), dtype=dtype, device="cuda")))
    have, at = r.positions >= 0, torch.where(r.positions >= 0, r.positions, 0).long()
    y64, w64, g64 = y.detach().double()[at] * have[:, :, None], w.detach().double(), g2.double()
    ref.check(back.detach(), (w64[:, :, None] * y64).sum(1), ref.sum_slack(k, (w64[:, :, None] * y64).abs().sum(1)), "combine")
    moved = g1.double()[at] * have[:, :, None]
    ref.check(dx, moved.sum(1), ref.sum_slack(k, moved.abs().sum(1)), "input gradient")
    slot_w = torch.where(used, w64.reshape(-1)[slot], 0.0)[:, None]
    ref.check(dy, slot_w * g64[slot // k], 2.0 ** -23 * (slot_w * g64[slot // k]).abs(), "rows' gradient")
    ref.check(dw, (y64 * g64[:, None]).sum(2), ref.sum_slack(channels, (y64 * g64[:, None]).abs().sum(2)), "weights' gradient")
    # one of the two gradients alone
    assert torch.equal(torch.autograd.grad(qmlp.combine(y.detach(), r), [w], g2)[0], dw)
    assert torch.equal(torch.autograd.grad(qmlp.combine(y, r._replace(weights=w.detach())), [y], g2)[0], dy)


def test_exchange_layouts(qmlp):
    r = qmlp.route(rand(66, (80, 6)), 2)
    base = rand(67, (160, 50), torch.bfloat16)
    for x in (base[:80, :48], base[:80, 1:49], base[::2, :48], rand(68, (48, 80), torch.bfloat16).t()):
        assert torch.equal(qmlp.dispatch(x, r), x[r.order.long() // 2])
    for y in (base[:, :48], base[:, 1:49]):
        assert torch.equal(qmlp.combine(y, r), qmlp.combine(y.contiguous(), r))
    wild = r._replace(order=torch.full_like(r.order, 2 ** 30), positions=torch.full_like(r.positions, 2 ** 30))    # what no router writes is skipped
    assert not qmlp.dispatch(base[:80], wild).any() and not qmlp.combine(base, wild).any()


# ---- products grouped by expert ------------------------------------------------------------------------------------------
def offsets_of(counts, first=0):
    return torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32, device="cuda")


def experts_case(qmlp, x, weight, offsets, bias, grad):
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    y = qmlp.expert_linear(leaves[0], leaves[1], offsets, leaves[2] if bias is not None else None)
    got = torch.autograd.grad(y, leaves, grad)
    exact = ref.expert_linear(x, weight, offsets, bias, grad)
    assert y.dtype == x.dtype
    ref.check(y.detach(), *exact[0], "output")
    for t, e, name in zip(got, exact[1:], ("input gradient", "weight gradient", "bias gradient")):
        assert t.dtype == x.dtype
        ref.check(t, *e, name)


SHAPES = [  # counts of rows, channels in, channels out
    ([1], 8, 8), ([1, 0, 1], 64, 64), ([5, 0, 3, 0], 16, 24), ([128], 64, 64), ([127, 1, 129, 256], 64, 128), ([130, 0, 0, 70, 64], 128, 64),
    ([300, 5], 200, 136), ([64, 64], 72, 264), ([33] * 40, 64, 64), ([1000, 1], 256, 256), ([513, 2000], 64, 64), ([3000], 32, 48), ([700, 20], 520, 300),
    ([2, 1, 3], 13, 5), ([200, 17], 77, 65), ([1500, 0, 300], 264, 320), ([600, 1029], 144, 392), ([700, 513], 200, 130), ([90], 1, 1), ([20000, 0, 3, 5000], 64, 64), ([128] * 300, 128, 128), ([40000], 80, 64), ([9000, 1, 0, 11000], 64, 96), ([10, 140], 31, 257), ([40, 0, 30], 130, 7),
]


@pytest.mark.parametrize("dtype", FLOATS[1:], ids=IDS.get)
@pytest.mark.parametrize("counts,n_in,n_out", SHAPES, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}e{sum(v)}r")
def test_expert_linear(qmlp, counts, n_in, n_out, dtype):
    rows, experts = sum(counts), len(counts)
    experts_case(qmlp, rand(70, (rows, n_in), dtype), rand(71, (experts, n_out, n_in), dtype, n_in ** -0.5), offsets_of(counts),
                 rand(72, (experts, n_out), dtype) if rows % 2 else None, rand(73, (rows, n_out), dtype))


@pytest.mark.parametrize("experts", [3, 37, 512, 513])
def test_expert_linear_ragged(qmlp, experts):
    """runs of all lengths in no order, one far longer than the others, many empty: sums of cut runs, experts by length"""
    counts = [int(c) for c in ints(110, (experts,), -20, 90).clamp(min=0)]
    counts[experts // 2] = 3000
    rows = sum(counts)
    experts_case(qmlp, rand(111, (rows, 40), torch.float16), rand(112, (experts, 24, 40), torch.float16, 0.2), offsets_of(counts),
                 rand(113, (experts, 24), torch.float16), rand(114, (rows, 24), torch.float16))


@pytest.mark.parametrize("n_in,n_out,bias", [(66, 264, True), (530, 12, False), (31, 200, True), (256, 136, True)])
def test_expert_linear_mostly_empty(qmlp, n_in, n_out, bias):
    """few rows among many experts: gradients of the others are zeros, whatever lay there, and their matrices are not read"""
    experts, dtype = 150, torch.float16
    counts = [0] * experts
    counts[0], counts[70], counts[71], counts[149] = 2, 130, 1, 3
    x, w, g = rand(111, (136, n_in), dtype), rand(112, (experts, n_out, n_in), dtype, n_in ** -0.5), rand(113, (136, n_out), dtype)
    b = rand(114, (experts, n_out), dtype) if bias else None
    experts_case(qmlp, x, w, offsets_of(counts), b, g)
    empty = torch.tensor([c == 0 for c in counts], device="cuda")
    leaves = [t.requires_grad_() for t in (x, torch.where(empty[:, None, None], float("nan"), w))]
    dx, dw = torch.autograd.grad(qmlp.expert_linear(*leaves, offsets_of(counts)), leaves, g)
    assert dx.isfinite().all() and dw.isfinite().all() and not dw[empty].any()


def test_expert_linear_many(qmlp):
    """as many experts as are supported, most of them without a row"""
    counts = [0] * 2048
    counts[5], counts[777], counts[2047] = 3, 200, 1
    experts_case(qmlp, rand(74, (204, 16), torch.float16), rand(75, (2048, 16, 16), torch.float16), offsets_of(counts), rand(76, (2048, 16), torch.float16),
                 rand(77, (204, 16), torch.float16))


def test_expert_linear_outside(qmlp):
    """rows before the first and behind the last expert are zeros and take no part in a gradient, whatever they hold"""
    x, g = rand(78, (500, 64), torch.float16), rand(79, (500, 48), torch.float16)
    x[:37], x[400:], g[:37], g[400:] = float("nan"), INF, INF, float("nan")
    w, b, offsets = rand(80, (3, 48, 64), torch.float16), rand(81, (3, 48), torch.float16), offsets_of([100, 0, 263], 37)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = qmlp.expert_linear(leaves[0], leaves[1], offsets, leaves[2])
    got = torch.autograd.grad(y, leaves, g)
    for t in (y[:37], y[400:], got[0][:37], got[0][400:]):
        assert not t.any()
    inner = [t.clone().requires_grad_() for t in (x[37:400], w, b)]
    want = qmlp.expert_linear(inner[0], inner[1], offsets - 37, inner[2])
    assert torch.equal(y[37:400], want)
    for a, e in zip((got[0][37:400], got[1], got[2]), torch.autograd.grad(want, inner, g[37:400])):
        assert torch.isfinite(a).all() and torch.equal(a, e)


@pytest.mark.parametrize("counts", [[70, 58, 200], [600, 700]])
def test_expert_linear_not_finite(qmlp, counts):
    """an expert's infinities and NaN stay its own"""
    x, g = rand(82, (sum(counts), 40), torch.bfloat16), rand(83, (sum(counts), 72), torch.bfloat16)
    w, offsets = rand(84, (len(counts), 72, 40), torch.bfloat16), offsets_of(counts)
    x[counts[0]:counts[0] + counts[1]] = INF
    g[counts[0]:counts[0] + counts[1]] = float("nan")
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y = qmlp.expert_linear(*leaves, offsets)
    dx, dw = torch.autograd.grad(y, leaves, g)
    exact = ref.expert_linear(x.detach()[:counts[0]], w.detach()[:1], offsets[:2], None, g[:counts[0]])
    for a, e in zip((y.detach()[:counts[0]], dx[:counts[0]], dw[:1]), exact):
        ref.check(a, *e, "the expert before")
    assert torch.isnan(dw[1]).all() and (len(counts) < 3 or torch.isfinite(dw[2]).all())


def test_expert_linear_layouts(qmlp):
    """rows apart or off a 16-byte boundary, transposed weights, expanded gradients, single rows"""
    base, offsets = rand(85, (260, 120), torch.float16), offsets_of([100, 0, 30])
    w = rand(86, (3, 80, 96), torch.float16)
    for x in (base[:130, :96], base[:130, 5:101], base[::2, 8:104], rand(87, (96, 130), torch.float16).t(), base[:1, :96].expand(130, 96)):
        experts_case(qmlp, x, w, offsets, None, rand(88, (130, 80), torch.float16))
    for weight in (rand(89, (3, 96, 80), torch.float16).transpose(1, 2), rand(90, (3, 80, 100), torch.float16)[:, :, 2:98]):
        experts_case(qmlp, base[:130, :96], weight, offsets, None, rand(91, (130, 100), torch.float16)[:, 3:83])
    experts_case(qmlp, base[:130, :96], w, offsets, rand(92, (3, 80), torch.float16), rand(93, (1, 80), torch.float16).expand(130, 80))
    experts_case(qmlp, base[:130, :96], w, offsets, rand(94, (1, 80), torch.float16).expand(3, 80), torch.ones((1, 1), dtype=torch.float16, device="cuda").expand(130, 80))


def test_expert_linear_offsets(qmlp):
    """offsets that are out of range or out of order give empty or shorter runs, never an access outside"""
    x, w, g = rand(95, (300, 32), torch.float16), rand(96, (5, 40, 32), torch.float16), rand(97, (300, 40), torch.float16)
    for bad in ([-5, 100, 50, 400, 200, 1000], [300, 200, 100, 0, 0, 0], [0, 300, 0, 300, 0, 300], [2 ** 31 - 1] * 6, [-2 ** 31] * 6):
        experts_case(qmlp, x, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), None, g)


def test_expert_linear_threads(qmlp):
    """the first call of a thread of its own: nothing has bound the device's context to it yet"""
    import threading
    x, w, offsets, got = rand(98, (40, 16), torch.float16), rand(99, (2, 24, 16), torch.float16), offsets_of([25, 15]), []
    thread = threading.Thread(target=lambda: got.append(qmlp.expert_linear(x, w, offsets)))
    thread.start()
    thread.join()
    assert torch.equal(got[0], qmlp.expert_linear(x, w, offsets))


def test_expert_linear_empty(qmlp):
    x, w, b = (torch.ones(s, dtype=torch.float16, device="cuda", requires_grad=True) for s in ((0, 16), (3, 8, 16), (3, 8)))
    y = qmlp.expert_linear(x, w, offsets_of([0, 0, 0]), b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones((0, 8), dtype=torch.float16, device="cuda"))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not dw.any() and not db.any()


def test_expert_linear_difference(qmlp):
    """linear in each of its arguments: moved by a direction, the output moves by what the gradient says"""
    counts = [40, 90]
    args = [rand(100, (130, 32), torch.float16), rand(101, (2, 24, 32), torch.float16, 0.2), rand(102, (2, 24), torch.float16)]
    offsets, g = offsets_of(counts), rand(103, (130, 24), torch.float16)
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(qmlp.expert_linear(leaves[0], leaves[1], offsets, leaves[2]), leaves, g)
    for i in range(3):
        d = rand(104 + i, tuple(args[i].shape), torch.float16)
        moved = list(args)
        moved[i] = args[i] + d
        step = moved[i].double() - args[i].double()      # what the sum really moved by
        delta = qmlp.expert_linear(moved[0], moved[1], offsets, moved[2]).double() - qmlp.expert_linear(args[0], args[1], offsets, args[2]).double()
        out = [qmlp.expert_linear(a[0], a[1], offsets, a[2]).double().abs() for a in (args, moved)]
        bound = (g.double().abs() * (out[0] + out[1])).sum() * 2.0 ** -11 + (grads[i].double() * step).abs().sum() * 2.0 ** -11
        assert abs((delta * g.double()).sum() - (grads[i].double() * step).sum()) <= bound * 1.01


# ---- streams, graphs, modules, refusals --------------------------------------------------------------------------------------
def everything(qmlp, tokens, table, w, b, router, weight):
    x = qmlp.layer_norm(qmlp.embedding(tokens, table, 2.0), w, b)
    r = qmlp.route(x.float() @ router, 2)
    return qmlp.combine(qmlp.expert_linear(qmlp.dispatch(x, r), weight, r.offsets), r)


def test_streams_and_graphs(qmlp):
    """on a stream of the caller's, and replayed from a CUDA graph: the same bits as on the default stream"""
    args = [ints(110, (700,), 0, 50), rand(111, (50, 64), torch.float16), rand(112, (64,)), rand(113, (64,)), rand(114, (64, 8)), rand(115, (8, 48, 64), torch.float16, 0.1)]
    leaves = [a.clone().requires_grad_() if a.is_floating_point() else a for a in args]
    grads_of = [t for t in leaves if t.requires_grad]
    g = rand(116, (700, 48), torch.float16)
    y = everything(qmlp, *leaves)
    want = [y.detach()] + list(torch.autograd.grad(y, grads_of, g))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = everything(qmlp, *leaves)
        got = [y.detach()] + list(torch.autograd.grad(y, grads_of, g))
    side.synchronize()
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    with torch.no_grad(), torch.cuda.stream(side):
        everything(qmlp, *args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = everything(qmlp, *args)
    for _ in range(2):
        args[0].copy_(ints(117 + _, (700,), 0, 50))
        graph.replay()
        with torch.no_grad():
            assert torch.equal(out, everything(qmlp, *args))


def test_once_differentiable(qmlp):
    x = rand(120, (10, 8)).requires_grad_()
    dx, = torch.autograd.grad(qmlp.layer_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable"):
        dx.sum().backward()


def test_modules(qmlp):
    """codes, norm and experts trained together in front of a fused network: the loss falls"""
    import specs
    torch.manual_seed(0)
    net = qmlp.FusedNetwork(json.dumps(specs.identity_net(16, [32, 1], ["relu", "identity"])), weight_dtype=torch.float32)
    codes, norm = qmlp.FusedEmbedding(10, 16), qmlp.FusedLayerNorm(16)
    layer = qmlp.FusedExperts(16, 64, 16, experts=4, k=2)
    params = [p for m in (net, codes, norm, layer) for p in m.parameters()]
    opt = torch.optim.Adam(params, lr=1e-2)
    tokens, target = ints(121, (4096,), 0, 10), None
    target = torch.sin(tokens.float() * 1.7)[:, None]
    losses = []
    for _ in range(60):
        y = net(layer(norm(codes(tokens))).float())
        loss = torch.nn.functional.mse_loss(y, target)
        opt.zero_grad()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in params if p.requires_grad)
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.2 * losses[0], losses


def test_example():
    """the example's model, from coordinates to colour: its error falls"""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "images_by_experts.py")
    spec = importlib.util.spec_from_file_location("images_by_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses = module.fit(images=4, points=8192, steps=80, report=None)
    assert losses[-1] < 0.25 * losses[0], losses[::10]


def test_refusals(qmlp):
    from qmlp._capi import QmlpError
    x, h = rand(130, (10, 16)), rand(131, (10, 16), torch.float16)
    r = qmlp.route(rand(132, (10, 4)), 2)
    w = rand(133, (4, 8, 16), torch.float16)
    wrong = [
        lambda: qmlp.layer_norm(x.double()), lambda: qmlp.layer_norm(x, torch.ones(15, device="cuda")), lambda: qmlp.layer_norm(x, torch.ones(16, device="cuda").half()),
        lambda: qmlp.layer_norm(x, None, None, -1.0), lambda: qmlp.layer_norm(x.cpu()), lambda: qmlp.layer_norm(x, torch.ones(16)), lambda: qmlp.layer_norm(x[:, :0]),
        lambda: qmlp.layer_norm(x.int()), lambda: qmlp.embedding(r.weights, x), lambda: qmlp.embedding(r.experts, x[0]), lambda: qmlp.embedding(r.experts.short(), x),
        lambda: qmlp.embedding(r.experts, x.double()), lambda: qmlp.route(x, 0), lambda: qmlp.route(x, 17), lambda: qmlp.route(rand(134, (3, 1025)), 1),
        lambda: qmlp.route(x[0], 1), lambda: qmlp.dispatch(x[:9], r), lambda: qmlp.dispatch(x, r._replace(order=r.order.long())),
        lambda: qmlp.dispatch(x, r._replace(order=r.order[1:])), lambda: qmlp.combine(x, r), lambda: qmlp.combine(rand(135, (20, 4)), r._replace(weights=r.weights[1:])),
        lambda: qmlp.combine(rand(135, (20, 4)), r._replace(weights=r.weights.half())), lambda: qmlp.expert_linear(x, w, r.offsets), lambda: qmlp.expert_linear(x, w.float(), r.offsets),
        lambda: qmlp.expert_linear(h, w.bfloat16(), r.offsets), lambda: qmlp.expert_linear(h, w[:, :, :8], r.offsets), lambda: qmlp.expert_linear(h, w, r.offsets[1:]),
        lambda: qmlp.expert_linear(h, w, r.offsets.long()), lambda: qmlp.expert_linear(h, w, r.offsets, w[:, 0, :7]), lambda: qmlp.expert_linear(h, w[0], r.offsets),
        lambda: qmlp.expert_linear(h, w, r.offsets, w[:, :, 0].float()), lambda: qmlp.expert_linear(h, torch.empty((2049, 1, 16), dtype=torch.float16, device="cuda"),
                                                                                                     torch.zeros(2050, dtype=torch.int32, device="cuda")),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(QmlpError):
            call()
            print("not refused:", i)
    from qmlp import bindings
    net = bindings.Network(json.dumps({"num_inputs": 1, "num_outputs": 1, "activation_specification": ["qmlp/builtin-activations.json"],
                                       "encodings": [{"id": "Identity", "start_in": 0, "n_in": 1}], "network": [{"n_out": 1, "bias": False, "activation": "relu"}]}))
    with pytest.raises(QmlpError):      # the networks' own types are as they were
        net.inference(rand(136, (4, 1), torch.bfloat16), net.create_inference_parameters())
