"""4-bit layers as a program calls them: cast as a whole, with matrices of any magnitude."""
import pytest
import torch

import mx_reference as mx
import rows_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qmlp():
    import qmlp
    return qmlp


def rand(seed, shape, dtype=torch.float32, std=1.0):
    return (torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["half", "bfloat16"])
def test_served_layers_are_cast(qmlp, dtype):
    """to float32 and back to the products' type the biases are the same; another type rounds them and the router, and nothing else"""
    torch.manual_seed(1)
    layer = qmlp.FusedExperts(48, 96, 24, experts=4, dtype=dtype)
    with torch.no_grad():
        layer.bias1.uniform_(-1, 1)
        layer.bias2.uniform_(-1, 1)
    x = rand(2, (300, 48))
    with torch.no_grad():
        want = layer.quantized()(x)
        assert torch.equal(layer.quantized().float()(x), want) and torch.equal(layer.quantized().double()(x), want)
        for cast in (torch.float16, torch.bfloat16):
            for name in ("router", "bias1", "bias2"):
                getattr(layer, name).copy_(getattr(layer, name).to(cast).to(dtype).to(cast))
            assert torch.equal(layer.quantized().to(cast)(x), layer.quantized()(x))


def test_layers_in_64_bits_are_served(qmlp):
    torch.manual_seed(3)
    layer = qmlp.FusedExperts(48, 96, 24, experts=4)
    x = rand(4, (100, 48))
    with torch.no_grad():
        assert torch.equal(layer.double().quantized()(x), layer.float().quantized()(x))


def gradient_case(qmlp, w, grad, offsets=None):
    """the input gradient against the formula in 64 bits, with fp32 sums' slack; w (matrices, channels out, channels in), or one without offsets"""
    exact = mx.nearest(w).view(-1, *w.shape[-2:])
    leaf = torch.zeros((grad.shape[0], w.shape[-1]), dtype=grad.dtype, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(qmlp.mx_linear(leaf, qmlp.mx_quantize(w), offsets), leaf, grad)
    want, slack = mx.mx_linear(leaf.detach(), exact, offsets, None, grad)[1]
    want = in_range(want, grad.dtype)
    ref.check(dx, want, slack, "input gradient")
    return dx, want


def in_range(exact, dtype):
    """what lies beyond the type's largest number is rounded to an infinity"""
    return torch.where(torch.isinf(exact.to(dtype)), exact.to(dtype).to(ref.F64), exact)


def powers(low, high, shape, seed):
    """a power of two per block of 32 channels"""
    e = torch.randint(low, high + 1, (*shape[:-1], (shape[-1] + 31) // 32), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return mx.power_of_two(e).repeat_interleave(32, -1)[..., :shape[-1]].float()


@pytest.mark.parametrize("n_in,n_out,rows", [(40, 24, 3), (96, 200, 300), (777, 130, 60), (1024, 520, 700)])
@pytest.mark.parametrize("low,high,scale", [(-30, -30, 14), (-24, -24, 10), (18, 18, -12), (14, 14, -10), (-20, 0, 4), (-12, 12, -4), (-33, 0, 0), (-36, 3, 0), (-60, 4, 0), (-126, 6, -4), (100, 100, -24),
                                            (-126, -126, 15)])
def test_gradient_scales(qmlp, n_in, n_out, rows, low, high, scale):
    """half rows: matrices whose powers of two half does not hold, for blocks of one magnitude and of many; rows of dy with zeros where the largest blocks are, large enough
    that what is left counts"""
    w = rand(10, (n_out, n_in)) * powers(low, high, (n_out, n_in), 11)
    grad = (rand(12, (rows, n_out)) * 2.0 ** scale).half()
    gradient_case(qmlp, w, grad)
    middle = (low + high) // 2
    if low < high:
        # every other channel out has the lower half of the powers; every other row of dy is large there and zero elsewhere
        w = rand(13, (n_out, n_in))
        w[::2] *= powers(low, middle, w[::2].shape, 14)
        w[1::2] *= powers(middle, high, w[1::2].shape, 15)
        grad = (rand(16, (rows, n_out)) * 2.0 ** scale).half()
        grad[::2, 1::2] = 0.0
        grad[::2, ::2] = (rand(17, grad[::2, ::2].shape) * 2.0 ** min(13, 2 - middle)).half()
        dx, want = gradient_case(qmlp, w, grad)
        if middle > -35:
            assert dx[::2].any()


def test_gradient_scales_apart(qmlp):
    """blocks that lie 2^40 apart: what the small ones give is not lost, to the last bit where sums are exact; blocks of zeros and of NaN next to them"""
    n_in, n_out, rows = 160, 64, 40
    small, large = 2.0 ** -30, 2.0 ** 10
    level = torch.tensor([1.0, 2.0, -1.0, 4.0], device="cuda")
    number = torch.randint(4, (n_out, n_in), device="cuda", generator=torch.Generator(device="cuda").manual_seed(20))
    w = level[number]
    w[:, ::32] = 4.0
    w[:32] *= small
    w[32:] *= large
    w[:, 64:96] = 0.0
    grad = torch.zeros((rows, n_out), dtype=torch.float16, device="cuda")
    grad[::2, :32], grad[1::2, 32:] = 2.0 ** 12, 2.0 ** -10
    dx, want = gradient_case(qmlp, w, grad)
    assert torch.equal(dx.double(), want) and dx[::2].any() and not dx[:, 64:96].any()
    w[3, 130] = float("nan")
    leaf = torch.zeros((rows, n_in), dtype=torch.float16, device="cuda", requires_grad=True)
    bad, = torch.autograd.grad(qmlp.mx_linear(leaf, qmlp.mx_quantize(w)), leaf, grad)
    assert torch.isnan(bad[:, 128:]).all() and torch.equal(bad[:, :128], dx[:, :128])


@pytest.mark.parametrize("counts", [[3, 0, 200, 1, 0, 77], [1000, 900, 0, 700, 513, 1]])
def test_gradient_scales_of_experts(qmlp, counts):
    """each matrix has its own power; some of them far apart in themselves; rows of no expert, rows apart, both gradients together"""
    e, n_in, n_out, rows = len(counts), 264, 140, sum(counts) + 20
    offsets = torch.tensor([7 + sum(counts[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
    base = rand(21, (e, n_out, n_in))
    w = base * torch.tensor([2.0 ** p for p in (-40, 3, 0, 22, -3, -18)], device="cuda")[:, None, None]
    w[2, ::3] *= powers(-50, 0, w[2, ::3].shape, 22)
    w[5] *= powers(-30, 10, w[5].shape, 23)
    scale = torch.ones(rows, device="cuda")
    for i, s in enumerate((14, 0, 3, -16, 0, 4)):
        scale[offsets[i]:offsets[i + 1]] = 2.0 ** s
    grad = (rand(24, (rows, n_out + 3)) * scale[:, None]).half()[:, 1:n_out + 1]
    dx, want = gradient_case(qmlp, w, grad, offsets)
    assert not dx[:7].any() and not dx[-13:].any()
    q, bias = qmlp.mx_quantize(w), torch.zeros((e, n_out), dtype=torch.float16, device="cuda", requires_grad=True)
    leaf = torch.zeros((rows, n_in), dtype=torch.float16, device="cuda", requires_grad=True)
    both = torch.autograd.grad(qmlp.mx_linear(leaf, q, offsets, bias), [leaf, bias], grad)
    assert torch.equal(torch.isnan(both[0]), torch.isnan(dx)) and torch.equal(torch.nan_to_num(both[0]), torch.nan_to_num(dx))      # (infinities of dy among them)
    db, slack = mx.mx_linear(leaf.detach(), mx.nearest(w), offsets, None, grad)[2]
    ref.check(both[1], in_range(db, torch.float16), slack, "bias gradient")


def test_gradient_scales_bfloat16(qmlp):
    """bfloat16 holds every power"""
    for low, high, scale in ((-126, -126, 100), (100, 100, -90), (-60, 60, -20)):
        w = rand(30, (130, 320)) * powers(low, high, (130, 320), 31)
        gradient_case(qmlp, w, (rand(32, (150, 130)) * 2.0 ** scale).bfloat16())


def test_gradient_scales_captured(qmlp):
    """captured and replayed on other matrices: which way they go is found out in every replay"""
    n_in, n_out, rows = 96, 64, 100
    grad = rand(40, (rows, n_out), torch.float16)
    sets = [qmlp.mx_quantize(w) for w in (rand(41, (n_out, n_in)), rand(42, (n_out, n_in)) * 2.0 ** -28, rand(43, (n_out, n_in)) * powers(-60, 3, (n_out, n_in), 44))]
    codes, scales = sets[0].codes.clone(), sets[0].scales.clone()

    def adjoint(c, s):
        return torch.ops.qmlp_b200.mx_linear_adjoint(grad, c, s, n_in, None, True, False)[0]
    want = [adjoint(q.codes, q.scales) for q in sets]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = adjoint(codes, scales)
    for i in (0, 1, 2, 0, 2, 1):
        codes.copy_(sets[i].codes)
        scales.copy_(sets[i].scales)
        graph.replay()
        assert torch.equal(dx, want[i])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["half", "bfloat16"])
@pytest.mark.parametrize("n_in", [256, 130])
def test_gradient_leaves_matrices_without_rows(qmlp, dtype, n_in):
    """matrices of experts without rows are not decoded: most of the scratch memory is as it was; offsets out of order count as they are used"""
    import ctypes as C
    from qmlp import _capi
    lib, e, n_out, rows = _capi.lib(), 64, 200, 30
    w = rand(50, (e, n_out, n_in))
    q, grad = qmlp.mx_quantize(w), rand(51, (rows, n_out), dtype)
    m = _capi.Mx(matrices=e, rows=n_out, channels=n_in, codes=q.codes.data_ptr(), scales=q.scales.data_ptr())

    def view(t):
        v = _capi.Tensor(data=t.data_ptr(), precision=_capi.QMLP_HALF if t.dtype == torch.float16 else _capi.QMLP_BFLOAT16, ndim=2)
        v.sizes[0], v.sizes[1], v.strides[0], v.strides[1] = *t.shape, *t.stride()
        return C.byref(v)
    size = C.c_size_t()
    assert lib.qmlp_mx_linear_adjoint_memory(view(grad), C.byref(m), 1, C.byref(size)) == 0
    for used in ([0] * 6 + [10] * 40 + [30] * 19, [5] * 3 + [12] * 20 + [-1] * 20 + [7] * 20 + [99] * 2, [0] * 65, [-5] * 64 + [30]):
        offsets = torch.tensor(used, dtype=torch.int32, device="cuda")
        scratch = torch.full((size.value,), 0xA5, dtype=torch.uint8, device="cuda")
        dx = torch.full((rows, n_in), 7.0, dtype=dtype, device="cuda")
        assert lib.qmlp_mx_linear_adjoint(view(grad), C.byref(m), C.c_void_p(offsets.data_ptr()), view(dx), None, _capi.current_stream(), scratch.data_ptr(), size.value) == 0
        want, slack = mx.mx_linear(torch.zeros((rows, n_in), dtype=dtype, device="cuda"), mx.nearest(w), offsets, None, grad)[1]
        ref.check(dx, want, slack, "input gradient")
        rising = sum(min(max(b, 0), rows) > min(max(a, 0), rows) for a, b in zip(used, used[1:]))
        # what is written: their matrices, once more with padded rows where the channels ask for it, and what goes with rows and experts alone
        bound = rising * n_out * 2 * (n_in + (n_in + 7) // 8 * 8 if n_in % 8 else n_in) + rows * (n_out + 8) * 2 + e * 32 + 4096
        assert int((scratch != 0xA5).sum()) <= bound < size.value // 4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["half", "bfloat16"])
def test_gradient_of_odd_widths(qmlp, dtype):
    """matrices of any width are decoded once, to rows of a multiple of 8 channels: no more memory than for that multiple; what lies behind a row counts for nothing"""
    import ctypes as C
    from qmlp import _capi
    lib, e, n_out, rows = _capi.lib(), 5, 72, 700
    offsets, grad = torch.tensor([0, 100, 100, 420, 699, 700], dtype=torch.int32, device="cuda"), rand(60, (rows, n_out), dtype)
    view = _capi.Tensor(data=grad.data_ptr(), precision=_capi.QMLP_HALF if dtype == torch.float16 else _capi.QMLP_BFLOAT16, ndim=2)
    view.sizes[0], view.sizes[1], view.strides[0], view.strides[1] = rows, n_out, n_out, 1

    def memory(n_in):
        size, m = C.c_size_t(), _capi.Mx(matrices=e, rows=n_out, channels=n_in, codes=grad.data_ptr(), scales=grad.data_ptr())
        assert lib.qmlp_mx_linear_adjoint_memory(C.byref(view), C.byref(m), 1, C.byref(size)) == 0
        return size.value
    for n_in in (1, 7, 9, 33, 63, 65, 127, 130, 255, 777):
        assert memory(n_in) == memory((n_in + 7) // 8 * 8)
        gradient_case(qmlp, rand(61 + n_in, (e, n_out, n_in)), grad, offsets)


@pytest.mark.parametrize("power", [-40, -23, -22, -20, -17, -14, -13, 0, 13, 14, 20])
def test_gradient_sums_keep_their_bits(qmlp, power):
    """large terms cancel and leave small ones, which count whatever the matrix' magnitude: sums of whole numbers of units, up to 2^21 of them, exact in fp32"""
    n_in, rows = 64, 130
    w = torch.zeros((4, n_in), device="cuda")
    w[0], w[1], w[2], w[3] = 4.0, 4.0, 0.5, 1.0
    w[2, ::32] = w[3, ::32] = 4.0      # (every block has the power `power`)
    w = w * 2.0 ** power
    unit = 2.0 ** min(max(-7, -power - 4), 4)
    grad = torch.tensor([[1024.0, -1024.0, 3 / 256, 5 / 256]], device="cuda").expand(rows, 4) * unit
    grad = grad.half()
    assert (grad[0].abs() >= 2.0 ** -14).all()      # (normal numbers)
    dx, want = gradient_case(qmlp, w, grad)
    assert torch.equal(dx.double(), want.half().double())
