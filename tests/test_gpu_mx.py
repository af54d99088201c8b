"""4-bit matrices and their products against the definitions (mx_reference.py): every bit of codes and scales, types, odd sizes, strides, rows of no expert, NaN,
gradients, streams, graphs, refusals."""
import pytest
import torch

import mx_reference as mx
import rows_reference as ref

pytestmark = pytest.mark.gpu
FLOATS = [torch.float32, torch.float16, torch.bfloat16]
IDS = {torch.float32: "float", torch.float16: "half", torch.bfloat16: "bfloat16"}
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(dtype)


def same(a, e):
    """equal, NaN where NaN is due"""
    assert a.shape == e.shape and torch.equal(torch.isnan(a), torch.isnan(e))
    assert torch.equal(torch.nan_to_num(a.to(ref.F64), nan=0.0, posinf=1e300, neginf=-1e300), torch.nan_to_num(e.to(ref.F64), nan=0.0, posinf=1e300, neginf=-1e300))


def quantize_case(qmlp, x):
    q = qmlp.mx_quantize(x)
    number, exponent = mx.quantize(x)
    codes, scales = mx.pack(number, exponent)
    assert q.channels == x.shape[-1]
    assert torch.equal(q.scales, scales)
    assert torch.equal(q.codes, codes)
    exact = mx.values(number, exponent)[..., :x.shape[-1]]
    for dtype in FLOATS:
        same(qmlp.mx_dequantize(q, dtype), exact.to(dtype))
    return q


# ---- quantisation ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (1, 32), (3, 33), (5, 64), (127, 65), (128, 96), (129, 128), (300, 129), (257, 1000), (2, 5003), (1, 1024),
                                   (1, 5, 40), (3, 130, 77), (4, 128, 128), (2, 1, 20000)])
def test_quantize(qmlp, shape, dtype):
    scale = torch.exp(2 * rand(1, (*shape[:-1], 1)))
    quantize_case(qmlp, (rand(2, shape) * scale).to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
def test_quantize_every_value(qmlp, dtype):
    """all 65536 bit patterns, alone in their block, next to a larger and a smaller value, and the neighbours of borders and ties among them"""
    v = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)[:, None]
    x = torch.cat([v, torch.zeros_like(v).expand(-1, 31), v, torch.full_like(v, 4.0), torch.zeros_like(v).expand(-1, 30), v.expand(-1, 3), torch.full_like(v, 2.0 ** -10).expand(-1, 29)], 1)
    quantize_case(qmlp, x)


def test_quantize_float_borders(qmlp):
    """fp32 numbers at and next to every border between codes, at scales from the smallest to the largest"""
    borders = torch.tensor([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0, 7.9999995], device="cuda", dtype=torch.float64)
    rows = []
    for power in (-149, -140, -128, -127, -126, -30, 0, 100, 125):
        unit = mx.power_of_two(torch.tensor(power, device="cuda"))
        b = (borders * unit).float()
        for n in (b, torch.nextafter(b, torch.zeros_like(b)), torch.nextafter(b, torch.full_like(b, INF))):
            rows.append(torch.cat([-n[torch.isfinite(n)], n[torch.isfinite(n)]]))
    x = torch.zeros((len(rows) * 32, 64), device="cuda")
    for i, n in enumerate(rows):
        for j in range(32):      # one of them with the block's largest, 7.99... or 4 of the unit, and alone
            x[i * 32 + j, :2] = torch.stack([n[j % n.numel()], n.abs().max()])
            x[i * 32 + j, 40] = n[j % n.numel()]
    quantize_case(qmlp, x)


def test_quantize_special(qmlp):
    """zeros of both signs, blocks with an infinity or NaN (theirs alone), numbers below the smallest scale, the largest"""
    x = rand(3, (140, 96))
    x[0], x[1], x[2, :32], x[3, 5], x[4, 40], x[5, 95] = 0.0, -0.0, -0.0, INF, NAN, -INF
    x[6], x[7], x[8], x[9, :32] = 2.0 ** -149, 2.0 ** -127, 3.4028234663852886e38, 1e-40
    q = quantize_case(qmlp, x)
    bad = torch.isnan(qmlp.mx_dequantize(q, torch.float32))
    assert bad.sum() == 96 and bad[3, :32].all() and bad[4, 32:64].all() and bad[5, 64:].all()


@pytest.mark.parametrize("dtype", FLOATS, ids=IDS.get)
def test_quantize_layouts(qmlp, dtype):
    base = rand(4, (300, 200), dtype)
    for x in (base[:, :96], base[:, 1:97], base[::2, 8:137], base.t(), base[:1, 3:99].expand(150, 96), base.view(3, 100, 200)[:, 10:60, 5:101], base.view(3, 100, 200).transpose(0, 1)):
        quantize_case(qmlp, x)
    q = qmlp.mx_quantize(base)
    odd = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(q.codes.shape).copy_(q.codes)      # off a 16-byte boundary
    spread = torch.stack([q.codes, q.codes], -1)[..., 0]
    for codes in (odd, spread):
        same(qmlp.mx_dequantize(q._replace(codes=codes), dtype), qmlp.mx_dequantize(q, dtype))


def test_quantize_empty(qmlp):
    for shape in ((0, 32), (0, 5, 40), (3, 0, 40)):
        q = qmlp.mx_quantize(torch.empty(shape, device="cuda"))
        assert q.codes.numel() == 0 and qmlp.mx_dequantize(q).shape == shape


# ---- products ---------------------------------------------------------------------------------------------------------------
def offsets_of(counts, first=0):
    return torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32, device="cuda")


def weights(qmlp, seed, shape):
    """a 4-bit tensor and its values in 64 bits (experts, channels out, channels in)"""
    w = rand(seed, shape, std=shape[-1] ** -0.5)
    return qmlp.mx_quantize(w), mx.nearest(w).view(-1, *shape[-2:])


def linear_case(qmlp, x, weight, exact, offsets, bias, grad=None):
    leaves = [t.detach().requires_grad_() if t is not None and grad is not None else t for t in (x, bias)]
    y = qmlp.mx_linear(leaves[0], weight, offsets, leaves[1])
    want = mx.mx_linear(x, exact, offsets, bias, grad)
    assert y.dtype == x.dtype
    ref.check(y.detach(), *want[0], "output")
    if grad is not None:
        got = torch.autograd.grad(y, [t for t in leaves if t is not None], grad)
        ref.check(got[0], *want[1], "input gradient")
        if bias is not None:
            ref.check(got[1].view(want[2][0].shape), *want[2], "bias gradient")
    return y.detach()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 1, 1), (1, 32, 8), (3, 33, 65), (1, 4096, 264), (5, 100, 4100), (64, 64, 64), (65, 256, 128), (129, 257, 129), (128, 320, 256), (200, 448, 72),
                                             (300, 1000, 300), (513, 512, 512), (1000, 96, 520), (2000, 777, 257), (1100, 2049, 258), (4097, 64, 48), (700, 5000, 24)])
def test_linear(qmlp, rows, n_in, n_out, dtype):
    """one matrix: every shape of tile, steps that are cut, single rows"""
    q, exact = weights(qmlp, 10, (n_out, n_in))
    linear_case(qmlp, rand(11, (rows, n_in), dtype), q, exact, None, rand(12, (n_out,), dtype), rand(13, (rows, n_out), dtype))
    linear_case(qmlp, rand(14, (rows, n_in), dtype), q, exact, None, None)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("counts,n_in,n_out", [([1, 1], 1024, 200), ([0, 5, 0, 3, 1], 100, 130), ([130, 0, 7, 128, 300], 64, 64), ([1, 127, 129, 255, 257], 160, 100),
                                               ([700, 600, 0, 900], 300, 520), ([257, 1500, 1], 256, 1000), ([64] * 40, 32, 24), ([3] * 300, 48, 300)])
def test_linear_experts(qmlp, counts, n_in, n_out, dtype):
    e, rows = len(counts), sum(counts)
    q, exact = weights(qmlp, 20, (e, n_out, n_in))
    linear_case(qmlp, rand(21, (rows, n_in), dtype), q, exact, offsets_of(counts), rand(22, (e, n_out), dtype), rand(23, (rows, n_out), dtype))


def test_linear_many(qmlp):
    """as many experts as are supported, most of them without a row"""
    counts = [0] * 2048
    counts[5], counts[777], counts[2047] = 3, 200, 1
    q, exact = weights(qmlp, 30, (2048, 16, 40))
    linear_case(qmlp, rand(31, (204, 40), torch.float16), q, exact, offsets_of(counts), rand(32, (2048, 16), torch.float16), rand(33, (204, 16), torch.float16))


def test_linear_outside(qmlp):
    """rows before the first and behind the last expert are zeros and take no part in a gradient, whatever they hold; offsets out of range or out of order"""
    q, exact = weights(qmlp, 40, (3, 48, 64))
    x, g, b, offsets = rand(41, (500, 64), torch.float16), rand(42, (500, 48), torch.float16), rand(43, (3, 48), torch.float16), offsets_of([100, 0, 263], 37)
    x[:37], x[400:], g[:37], g[400:] = NAN, INF, INF, NAN
    leaf = x.clone().requires_grad_()
    y = qmlp.mx_linear(leaf, q, offsets, b)
    dx, = torch.autograd.grad(y, leaf, g)
    for t in (y[:37], y[400:], dx[:37], dx[400:]):
        assert not t.any()
    want = linear_case(qmlp, x[37:400], q, exact, offsets - 37, b, g[37:400])
    assert torch.equal(y[37:400], want)
    x, g = rand(44, (300, 64), torch.float16), rand(45, (300, 48), torch.float16)
    for bad in ([-5, 100, 50, 400], [300, 200, 100, 0], [0, 300, 0, 300], [2 ** 31 - 1] * 4, [-2 ** 31] * 4):
        linear_case(qmlp, x, q, exact, torch.tensor(bad, dtype=torch.int32, device="cuda"), b, g)


@pytest.mark.parametrize("rows", [7, 40, 64])
def test_linear_few_rows_offsets(qmlp, rows):
    """a handful of rows: experts without rows, rows of nobody, offsets out of range or out of order, one expert with offsets"""
    q, exact = weights(qmlp, 46, (4, 72, 100))
    x, b, g = rand(47, (rows, 100), torch.float16), rand(48, (4, 72), torch.float16), rand(49, (rows, 72), torch.float16)
    for bad in ([0, 3, 3, 5, rows], [2, 2, 4, 4, 5], [-5, 6, 4, 5, 3], [rows, 3, 2, 1, 0], [0, rows, 0, rows, 0], [2 ** 31 - 1] * 5, [-2 ** 31] * 5, [-1, 1, 2, 3, 10 * rows], [1, 1, 1, 1, 1]):
        linear_case(qmlp, x, q, exact, torch.tensor(bad, dtype=torch.int32, device="cuda"), b, g)
    one = q._replace(codes=q.codes[:1], scales=q.scales[:1])
    for ends in ([0, rows], [2, 5], [3, 1], [0, 0]):
        linear_case(qmlp, x, one, exact[:1], torch.tensor(ends, dtype=torch.int32, device="cuda"), b[:1], g)


def test_linear_long(qmlp):
    """codes that pass 2^32 bytes: rows at both ends"""
    rows, n_in = 600000, 16384
    base = rand(52, (3, n_in), torch.float16)
    q, exact = weights(qmlp, 53, (40, n_in))
    offsets = None
    for at in (0, 2):
        y = qmlp.mx_linear(base[at:at + 1].expand(rows, n_in), q, offsets)
        want, slack = mx.mx_linear(base[at:at + 1], exact, None, None)[0]
        for r in (0, 131072, 262143, 524289, rows - 1):
            ref.check(y[r:r + 1], want, slack, f"row {r}")
        assert torch.equal(y[1:], y[:-1])


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 96, 40), (9, 96, 40), (200, 96, 40), (700, 300, 300)])
def test_linear_not_finite(qmlp, rows, n_in, n_out):
    """an infinity or NaN in a row makes that row NaN, one in a row of the matrix that channel, and nothing else"""
    w, x = rand(50, (n_out, n_in)), rand(51, (rows, n_in), torch.bfloat16)
    w[7, 3], w[n_out - 1, n_in - 1] = INF, NAN
    x[rows // 2, n_in - 2] = -INF
    y = qmlp.mx_linear(x, qmlp.mx_quantize(w))
    bad = torch.zeros((rows, n_out), dtype=torch.bool, device="cuda")
    bad[rows // 2], bad[:, 7], bad[:, n_out - 1] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    rows_of, columns_of = ~bad.all(1), ~bad.all(0)      # the others: as without
    if rows_of.any():
        want, slack = mx.mx_linear(x[rows_of], mx.nearest(w[columns_of])[None], None, None)[0]
        ref.check(y[rows_of][:, columns_of], want, slack, "the rest")


@pytest.mark.parametrize("rows", [1, 4, 33, 600])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS.get)
def test_linear_exact(qmlp, rows, dtype):
    """small numbers with few bits: every sum is exact in fp32 and in the result, and so is the product"""
    gen = torch.Generator(device="cuda").manual_seed(60)
    levels = torch.tensor([0.0, 1.0, -1.0, 2.0, -2.0, 4.0, -4.0, 0.5, -0.5], device="cuda")
    x = levels[torch.randint(9, (rows, 512), device="cuda", generator=gen)] * (torch.rand((rows, 512), device="cuda", generator=gen) < 0.02)
    w = levels[torch.randint(9, (300, 512), device="cuda", generator=gen)]
    x[:, ::32], w[:, ::32] = 4.0, 4.0      # every block's scale is 1
    x[:, ::64] *= -1
    y = qmlp.mx_linear(x.to(dtype), qmlp.mx_quantize(w))
    exact = x.double() @ w.double().T
    assert torch.equal(exact.to(dtype).double(), exact) or dtype == torch.bfloat16
    assert torch.equal(y, exact.to(dtype))


def test_linear_scales(qmlp):
    """blocks of very different magnitude next to one another, down to the smallest scale"""
    gen = torch.Generator(device="cuda").manual_seed(61)
    for rows, n_in, n_out in ((2, 256, 40), (150, 1056, 40), (600, 288, 300)):
        wide, w = (rand(62, (n, n_in)) * mx.power_of_two(torch.randint(-12, 12, (n, n_in // 32), device="cuda", generator=gen).repeat_interleave(32, 1)).float() for n in (rows, n_out))
        linear_case(qmlp, wide.bfloat16(), qmlp.mx_quantize(w), mx.nearest(w)[None], None, None)
        tiny = rand(64, (n_out, n_in)) * 2.0 ** -126
        linear_case(qmlp, (rand(65, (rows, n_in)) * 2.0 ** 100).bfloat16(), qmlp.mx_quantize(tiny), mx.nearest(tiny)[None], None, None)


def test_linear_layouts(qmlp):
    """rows apart or off a 16-byte boundary, transposed, expanded; more than two dimensions; codes and scales that have to be copied"""
    base, offsets = rand(70, (260, 120), torch.float16), offsets_of([100, 0, 30])
    q, exact = weights(qmlp, 71, (3, 80, 96))
    b = rand(72, (1, 80), torch.float16).expand(3, 80)
    for x in (base[:130, :96], base[:130, 5:101], base[::2, 8:104], rand(73, (96, 130), torch.float16).t(), base[:1, :96].expand(130, 96)):
        for g in (rand(74, (130, 100), torch.float16)[:, 3:83], torch.ones((1, 1), dtype=torch.float16, device="cuda").expand(130, 80)):
            linear_case(qmlp, x, q, exact, offsets, b, g)
    one = q._replace(codes=q.codes[1], scales=q.scales[1])      # views
    odd = q._replace(codes=torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(q.codes.shape).copy_(q.codes))
    want = linear_case(qmlp, base[:130, :96], q, exact, offsets, None)
    assert torch.equal(qmlp.mx_linear(base[:130, :96], odd, offsets), want)
    leaf = base[:120, :96].reshape(4, 5, 6, 96).clone().requires_grad_()
    y = qmlp.mx_linear(leaf, one)
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    flat = linear_case(qmlp, base[:120, :96], one, exact[1:2], None, None, torch.ones((120, 80), dtype=torch.float16, device="cuda"))
    assert y.shape == (4, 5, 6, 80) and torch.equal(y.view(120, 80), flat) and dx.shape == leaf.shape


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["half", "bfloat16"])
@pytest.mark.parametrize("counts,n_in,n_out", [(None, 40, 7), (None, 300, 130), ([3000, 0, 1, 2049], 512, 200), ([33, 31, 700], 96, 65), ([5] * 100, 130, 333), ([70000], 32, 66)])
def test_linear_gradients_apart(qmlp, counts, n_in, n_out, dtype):
    """the gradients of the rows, of the bias, and of both: each for itself what the formula says, and the rows' the same either way"""
    e, rows = (1, 777) if counts is None else (len(counts), sum(counts))
    q, exact = weights(qmlp, 85, (n_out, n_in) if counts is None else (e, n_out, n_in))
    x, b, g = rand(86, (rows, n_in), dtype), rand(87, (n_out,) if counts is None else (e, n_out), dtype), rand(88, (rows, n_out), dtype)
    offsets = None if counts is None else offsets_of(counts)
    want = mx.mx_linear(x, exact, offsets, b, g)
    got = []
    for rows_too, bias_too in ((True, True), (True, False), (False, True)):
        leaves = [x.clone().requires_grad_(rows_too), b.clone().requires_grad_(bias_too)]
        grads = list(torch.autograd.grad(qmlp.mx_linear(leaves[0], q, offsets, leaves[1]), [t for t in leaves if t.requires_grad], g))
        got.append(grads.pop(0) if rows_too else None)
        if rows_too:
            ref.check(got[-1], *want[1], "rows")
        if bias_too:
            ref.check(grads[0].view(want[2][0].shape), *want[2], "bias")
    assert torch.equal(got[0], got[1])


def test_linear_empty(qmlp):
    q, _ = weights(qmlp, 80, (3, 8, 16))
    x, b = (torch.ones(s, dtype=torch.float16, device="cuda", requires_grad=True) for s in ((0, 16), (3, 8)))
    y = qmlp.mx_linear(x, q, offsets_of([0, 0, 0]), b)
    dx, db = torch.autograd.grad(y, [x, b], torch.ones((0, 8), dtype=torch.float16, device="cuda"))
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not db.any()


def test_linear_difference(qmlp):
    """rows that are 4-bit numbers already, moved to others with the same scales: the output moves by what the gradient says, exactly"""
    gen = torch.Generator(device="cuda").manual_seed(90)
    q, exact = weights(qmlp, 91, (40, 96))
    x = torch.randint(-2, 3, (50, 96), device="cuda", generator=gen).half()
    x[:, ::32] = 4.0
    d = torch.randint(-1, 2, (50, 96), device="cuda", generator=gen).half()
    d[:, ::32] = 0.0
    g = torch.randint(-2, 3, (50, 40), device="cuda", generator=gen).half()
    leaf, bias = x.clone().requires_grad_(), rand(92, (40,), torch.float16).requires_grad_()
    dx, db = torch.autograd.grad(qmlp.mx_linear(leaf, q, None, bias), [leaf, bias], g)
    with torch.no_grad():
        outs = [qmlp.mx_linear(t, q, None, bias).double() for t in (x, x + d)]
    bound = sum((g.double().abs() * o.abs()).sum() for o in outs) * 2.0 ** -11 + (dx.double() * d.double()).abs().sum() * 2.0 ** -11
    assert abs(((outs[1] - outs[0]) * g.double()).sum() - (dx.double() * d.double()).sum()) <= bound * 1.01
    assert torch.equal(db, g.sum(0))


def test_linear_streams_and_graphs(qmlp):
    """another stream and thread; captured with its gradient; two graphs replayed in turn"""
    import threading
    q, _ = weights(qmlp, 100, (4, 300, 160))
    offsets, g = offsets_of([100, 500, 0, 100]), rand(101, (700, 300), torch.float16)
    leaf = rand(102, (700, 160), torch.float16).requires_grad_()

    def both():
        y = qmlp.mx_linear(leaf, q, offsets)
        return [y.detach(), *torch.autograd.grad(y, leaf, g)]
    want, got = both(), []
    thread = threading.Thread(target=lambda: got.extend(both()))
    thread.start()
    thread.join()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(both())
    for i in (0, 1, 1, 0):
        with torch.no_grad():
            leaf.copy_(rand(110 + i, (700, 160), torch.float16))
        graphs[i].replay()
        assert all(torch.equal(a, e) for a, e in zip(outs[i], both()))
    with torch.no_grad():
        leaf.copy_(rand(102, (700, 160), torch.float16))
    dx, = torch.autograd.grad(qmlp.mx_linear(leaf, q, offsets), leaf, g)
    assert torch.equal(dx, want[1])


def test_linear_repeats(qmlp):
    """the same bits every run, back to back on inputs in turn"""
    q, _ = weights(qmlp, 120, (2, 640, 520))
    offsets, xs = offsets_of([1000, 1100]), [rand(121 + i, (2100, 520), torch.bfloat16) for i in range(2)]
    want = [qmlp.mx_linear(x, q, offsets) for x in xs]
    for _ in range(20):
        for x, e in zip(xs, want):
            assert torch.equal(qmlp.mx_linear(x, q, offsets), e)


def test_refusals(qmlp):
    from qmlp._capi import QmlpError
    x, h = rand(130, (10, 40)), rand(131, (10, 40), torch.float16)
    q, _ = weights(qmlp, 132, (24, 40))
    e, _ = weights(qmlp, 133, (3, 24, 40))
    o, b = offsets_of([5, 3, 2]), rand(134, (24,), torch.float16)
    half = torch.float16
    wrong = [
        lambda: qmlp.mx_quantize(x.double()), lambda: qmlp.mx_quantize(x.int()), lambda: qmlp.mx_quantize(x.cpu()), lambda: qmlp.mx_quantize(x[0]),
        lambda: qmlp.mx_quantize(x[:, :0]), lambda: qmlp.mx_quantize(x[None, None]), lambda: qmlp.mx_dequantize(q, torch.float64), lambda: qmlp.mx_dequantize(q, torch.int32),
        lambda: qmlp.mx_dequantize(q._replace(channels=65)), lambda: qmlp.mx_dequantize(q._replace(channels=0)), lambda: qmlp.mx_dequantize(q._replace(codes=q.codes.int())),
        lambda: qmlp.mx_dequantize(q._replace(codes=q.codes[:, :16])), lambda: qmlp.mx_dequantize(q._replace(scales=q.scales[:, :0])),
        lambda: qmlp.mx_dequantize(q._replace(scales=q.scales.view(-1))), lambda: qmlp.mx_dequantize(q._replace(scales=e.scales)), lambda: qmlp.mx_dequantize(q._replace(scales=q.scales.cpu())),
        lambda: qmlp.mx_linear(x, q), lambda: qmlp.mx_linear(h.double(), q), lambda: qmlp.mx_linear(h[:, :39], q), lambda: qmlp.mx_linear(h.cpu(), q), lambda: qmlp.mx_linear(h, q, o),
        lambda: qmlp.mx_linear(h, e), lambda: qmlp.mx_linear(h, e, o[1:]), lambda: qmlp.mx_linear(h, e, o.long()), lambda: qmlp.mx_linear(h, e, o.cpu()), lambda: qmlp.mx_linear(h, q, None, b[1:]),
        lambda: qmlp.mx_linear(h, q, None, b.float()), lambda: qmlp.mx_linear(h, q, None, b[None]), lambda: qmlp.mx_linear(h, e, o, b), lambda: qmlp.mx_linear(h, e, o, b.expand(2, 24)),
        lambda: qmlp.mx_linear(h, q._replace(scales=q.scales.float())), lambda: qmlp.mx_linear(h[0, 0], q), lambda: qmlp.mx_linear(h[:, :0], q._replace(channels=0)),
        lambda: qmlp.mx_linear(h, qmlp.mx_quantize(torch.zeros((2049, 1, 40), dtype=half, device="cuda")), torch.zeros(2050, dtype=torch.int32, device="cuda")),
        lambda: qmlp.mx_linear(h, qmlp.mx_quantize(torch.zeros((0, 40), dtype=half, device="cuda"))),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(QmlpError):
            call()
            print("not refused:", i)
    y = qmlp.mx_linear(h.clone().requires_grad_(), q)
    dx, = torch.autograd.grad(y, y.grad_fn.next_functions[0][0].variable, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
