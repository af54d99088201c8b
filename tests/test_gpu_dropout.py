"""Dropout against its definition (mx_reference.py): the generator's bits, types, odd sizes, strides, gradients, streams, graphs, refusals."""
import pytest
import torch

import mx_reference as mx
import rows_reference as ref

pytestmark = pytest.mark.gpu
FLOATS = [torch.float32, torch.float16, torch.bfloat16]
IDS = {torch.float32: "float", torch.float16: "half", torch.bfloat16: "bfloat16"}
SEED, OFFSET = 0x123456789abcdef0, 0x1_0000_0002


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(dtype)


def kept(shape, p, seed=SEED, offset=OFFSET):
    n = 1
    for s in shape:
        n *= s
    return mx.kept(0, n, p, seed, offset).view(shape).cuda()


def case(qmlp, x, residual, p, grad, seed=SEED, offset=OFFSET):
    leaves = [t.detach().requires_grad_() for t in (x, residual) if t is not None]
    y = qmlp.dropout(leaves[0], p, seed, offset, residual=leaves[1] if residual is not None else None)
    assert y.dtype == x.dtype and y.shape == x.shape
    keep = kept(tuple(x.shape), p, seed, offset)
    ref.check(y.detach(), *mx.dropout(x, keep, p, residual), "output")
    got = torch.autograd.grad(y, leaves, grad)
    ref.check(got[0], *mx.dropout(grad, keep, p), "input gradient")
    if residual is not None:
        assert torch.equal(got[1], grad)
    return y


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("rows,channels", [(1, 1), (1, 7), (1, 8), (9, 1), (16, 64), (13, 7), (1000, 8), (517, 13), (3, 20001), (2050, 96), (70, 1032), (1, 300000)])
def test_dropout(qmlp, rows, channels, dtype):
    x, r, g = rand(1, (rows, channels), dtype, 1.5), rand(2, (rows, channels), dtype), rand(3, (rows, channels), dtype)
    case(qmlp, x, None, 0.1, g)
    case(qmlp, x, r, 0.5, g)


@pytest.mark.parametrize("seed,offset", [(0, 0), (-1, -1), (2 ** 63 - 1, 2 ** 32), (-2 ** 63, -2 ** 63), (1 << 32, (1 << 32) - 1)])
def test_dropout_numbers(qmlp, seed, offset):
    """seed and offset are 64 bits, both halves count"""
    x = rand(4, (33, 24))
    y = case(qmlp, x, None, 0.5, x, seed, offset)
    for other in ((seed ^ 1, offset), (seed ^ 1 << 40, offset), (seed, offset ^ 1), (seed, offset ^ 1 << 40)):
        assert not torch.equal(y, qmlp.dropout(x, 0.5, *other))


def test_dropout_step(qmlp):
    """the step on the device adds to the offset, modulo 2^64"""
    x = rand(5, (40, 24), torch.float16)
    for offset, step in ((3, 4), (3, -4), (2 ** 63 - 1, 2 ** 63 - 1), (-1, 2)):
        total = (offset + step + 2 ** 63) % 2 ** 64 - 2 ** 63
        leaf, t = x.clone().requires_grad_(), torch.tensor([step], device="cuda")
        y = qmlp.dropout(leaf, 0.3, SEED, offset, step=t)
        assert torch.equal(y, qmlp.dropout(x, 0.3, SEED, total))
        assert torch.equal(torch.autograd.grad(y, leaf, x)[0], qmlp.dropout(x, 0.3, SEED, total))
    assert torch.equal(qmlp.dropout(x, 0.3, SEED, 1, step=torch.tensor(2, device="cuda")), qmlp.dropout(x, 0.3, SEED, 3))
    y = qmlp.dropout(leaf, 0.3, SEED, 0, step=t)
    t.add_(1)      # the gradient would drop other elements
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, x)


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
def test_dropout_layouts(qmlp, dtype):
    """rows apart, off a 16-byte boundary, transposed, expanded: an element's number goes with its place"""
    base, r = rand(6, (300, 130), dtype), rand(7, (100, 96), dtype)
    want = None
    for x in (base[:100, :96], base[:100, 1:97], base[::3, 8:104], rand(8, (96, 100), dtype).t(), base[:1, :96].expand(100, 96), base[:100 * 96 // 130 + 1].reshape(-1)[5:5 + 9600].view(100, 96)):
        for residual in (None, r, base[100:200, 3:99], base[100:200, 16:112]):
            y = case(qmlp, x, residual, 0.25, rand(9, (100, 100), dtype)[:, 2:98])
        assert torch.equal(y, qmlp.dropout(x.contiguous(), 0.25, SEED, OFFSET, residual=base[100:200, 16:112].contiguous()))
        dropped = qmlp.dropout(torch.ones_like(x), 0.25, SEED, OFFSET) == 0
        want = dropped if want is None else want
        assert torch.equal(dropped, want)
    x = rand(10, (4, 5, 7, 24), dtype)
    assert torch.equal(qmlp.dropout(x, 0.4, 1), qmlp.dropout(x.view(140, 24), 0.4, 1).view(x.shape))
    case(qmlp, x.transpose(0, 2), None, 0.4, x.transpose(0, 2))


def test_dropout_probabilities(qmlp):
    """none, all, below and at half a unit of the 16 bits; dropped infinities and NaN are zeros; the share that is dropped"""
    x, r = rand(11, (500, 64)), rand(12, (500, 64))
    assert torch.equal(qmlp.dropout(x, 0.0, 5), x) and torch.equal(qmlp.dropout(x, 2.0 ** -18, 5), x)
    assert not qmlp.dropout(x, 1.0, 5).any() and torch.equal(qmlp.dropout(x, 1.0, 5, residual=r), r)
    leaf = x.clone().requires_grad_()
    assert not torch.autograd.grad(qmlp.dropout(leaf, 1.0, 5), leaf, r)[0].any()
    bad = torch.full_like(x, float("nan"))
    for residual in (r, r[:1].expand(500, 64), r.t().contiguous().t(), rand(16, (500, 70))[:, 3:67]):
        assert torch.equal(qmlp.dropout(bad, 1.0, 5, residual=residual), residual)
    assert not qmlp.dropout(bad[:, 1:50], 1.0, 5).any()
    case(qmlp, x, r, 1 - 2.0 ** -16, x)
    for bad in (float("inf"), float("nan")):
        y = qmlp.dropout(torch.full_like(x, bad), 0.5, SEED, OFFSET, residual=r)
        keep = kept((500, 64), 0.5)
        assert torch.equal(y[~keep], r[~keep]) and not torch.isfinite(y[keep]).any()
    n = 1 << 24      # independent numbers: five deviations of a binomial distribution
    share = (qmlp.dropout(torch.ones((n // 64, 64), dtype=torch.float16, device="cuda"), 0.1, 77) == 0).double().mean().item()
    p = round(0.1 * 65536) / 65536
    assert abs(share - p) < 5 * (p * (1 - p) / n) ** 0.5


def test_dropout_empty(qmlp):
    x = torch.empty((0, 32), device="cuda", requires_grad=True)
    y = qmlp.dropout(x, 0.1, 1, residual=torch.empty((0, 32), device="cuda"))
    assert y.shape == (0, 32) and torch.autograd.grad(y, x, y)[0].shape == (0, 32)


def test_dropout_many(qmlp):
    """more than 2^32 elements: their numbers at both ends, whichever way the rows are read"""
    rows, channels = 65600, 65544      # 4.3e9
    row = torch.ones((1, channels), dtype=torch.float16, device="cuda")
    y = qmlp.dropout(row.expand(rows, channels), 0.5, SEED, OFFSET)
    for at in (0, 32768, 65537, rows - 1):
        assert torch.equal(y[at] != 0, mx.kept(at * channels, channels, 0.5, SEED, OFFSET).cuda())
    y = qmlp.dropout(y, 0.5, SEED, OFFSET)      # (a contiguous input)
    for at in (0, 32768, 65537, rows - 1):
        assert torch.equal(y[at] != 0, mx.kept(at * channels, channels, 0.5, SEED, OFFSET).cuda())


def test_dropout_linear(qmlp):
    """differences: the output moves by exactly what the gradient says where the arithmetic is exact; differentiable twice"""
    x, d = torch.randint(-8, 9, (30, 40), device="cuda").float(), torch.randint(-8, 9, (30, 40), device="cuda").float()
    leaf = x.clone().requires_grad_()
    g = torch.randint(-8, 9, (30, 40), device="cuda").float().requires_grad_()
    y = qmlp.dropout(leaf, 0.5, SEED)      # (times 2)
    dx, = torch.autograd.grad(y, leaf, g, create_graph=True)
    delta = qmlp.dropout(x + d, 0.5, SEED) - qmlp.dropout(x, 0.5, SEED)
    assert (delta * g).sum() == (dx * d).sum()
    back, = torch.autograd.grad(dx, g, d)
    assert torch.equal(back, qmlp.dropout(d, 0.5, SEED))


def test_dropout_streams_and_graphs(qmlp):
    """on another stream; captured with its gradient, replayed with an advanced step: the bits of the eager calls"""
    x, g, step = rand(13, (200, 72), torch.float16), rand(14, (200, 72), torch.float16), torch.zeros(1, dtype=torch.int64, device="cuda")
    leaf = x.clone().requires_grad_()

    def both(step=None, offset=0):
        y = qmlp.dropout(leaf, 0.2, SEED, offset, step=step)
        return [y.detach(), *torch.autograd.grad(y, leaf, g)]
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(step)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(step)
        step.add_(1)
    for i in range(3):
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, both(offset=i)))
    assert all(torch.equal(a, e) for a, e in zip(both(), want))


def test_dropout_refusals(qmlp):
    from qmlp._capi import QmlpError
    x, step = rand(15, (10, 16)), torch.zeros(1, dtype=torch.int64, device="cuda")
    wrong = [lambda: qmlp.dropout(x.double(), 0.1, 1), lambda: qmlp.dropout(x.int(), 0.1, 1), lambda: qmlp.dropout(x.cpu(), 0.1, 1), lambda: qmlp.dropout(x, -0.1, 1),
             lambda: qmlp.dropout(x, 1.1, 1), lambda: qmlp.dropout(x, float("nan"), 1), lambda: qmlp.dropout(x, 0.1, 1, residual=x[:1]),
             lambda: qmlp.dropout(x, 0.1, 1, residual=x.half()), lambda: qmlp.dropout(x, 0.1, 1, residual=x.cpu()), lambda: qmlp.dropout(x, 0.1, 1, residual=x[:, 0]),
             lambda: qmlp.dropout(x, 0.1, 1, step=step.int()), lambda: qmlp.dropout(x, 0.1, 1, step=step.cpu()), lambda: qmlp.dropout(x, 0.1, 1, step=step.expand(2)),
             lambda: qmlp.dropout(x[:, :0], 0.1, 1), lambda: qmlp.dropout(x[0, 0], 0.1, 1)]
    for i, call in enumerate(wrong):
        with pytest.raises(QmlpError):
            call()
            print("not refused:", i)
    for seed in (2 ** 63, -2 ** 63 - 1):
        with pytest.raises(TypeError):
            qmlp.dropout(x, 0.1, seed)
