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


def test_expert_linear_few_rows_wide(qmlp):
    """few rows of every width around the shared memory that a block has without asking, in ascending order and a process of its own: a wider
    call before would have asked for it"""
    import os
    import subprocess
    import sys
    code = """
import torch, qmlp
torch.manual_seed(0)
for dtype in (torch.float16, torch.bfloat16):
    for n_in in (2816, 2824, 2880, 2944, 3041, 3056, 3064, 3071, 3080, 3328):
        for rows in (1, 5):
            x, w = (torch.randint(-2, 3, s, device="cuda").to(dtype) for s in ((rows, n_in), (3, 24, n_in)))
            for first in (0, 1):     # 16-byte and single accesses
                w = torch.randint(-2, 3, (3 * 24 * n_in + 1,), device="cuda").to(dtype)[first:first + 3 * 24 * n_in].view(3, 24, n_in)
                y = qmlp.expert_linear(x, w, torch.tensor([0, 1, 1, rows], dtype=torch.int32, device="cuda"))
                exact = torch.cat([x[:1].double() @ w[0].double().T, x[1:].double() @ w[2].double().T])
                assert torch.equal(y, exact.to(dtype)), (n_in, rows, first)
print("fine")
"""
    package = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "quick-mlp_b200")
    done = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": package}, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float", "bfloat16"])
def test_leading_dimensions(qmlp, dtype):
    """rows of more than two dimensions, (experts, capacity, channels) say: every operator's gradient has the shape of what it is a gradient of, and is the
    flat call's"""
    r = qmlp.route(rand(10, (30, 6)), 2)
    w = r.weights.clone().requires_grad_()
    y, x, g, gx = rand(11, (6, 10, 16), dtype), rand(12, (5, 6, 16), dtype), rand(13, (30, 16), dtype), rand(14, (60, 16), dtype)
    got, want = [], []
    for shape, out in ((lambda t: t, got), (lambda t: t.reshape(-1, 16), want)):
        rows, inputs = shape(y).clone().requires_grad_(), shape(x).clone().requires_grad_()
        back, sent = qmlp.combine(rows, r._replace(weights=w)), qmlp.dispatch(inputs, r)
        grads = torch.autograd.grad([back, sent], [rows, w, inputs], [g, gx])
        assert grads[0].shape == rows.shape and grads[2].shape == inputs.shape
        out += [back.detach(), sent.detach(), *(t.reshape(-1, t.shape[-1]) for t in grads)]
        only, = torch.autograd.grad(qmlp.combine(rows, r), [rows], g)
        assert only.shape == rows.shape and torch.equal(only, grads[0])
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    if dtype != torch.float32:
        h, weight, offsets = rand(15, (4, 15, 16), dtype).requires_grad_(), rand(16, (6, 24, 16), dtype).requires_grad_(), r.offsets
        dh, dw = torch.autograd.grad(qmlp.expert_linear(h, weight, offsets), [h, weight], rand(17, (60, 24), dtype))
        assert dh.shape == h.shape and dw.shape == weight.shape


@pytest.mark.parametrize("rows", [1, 37, 5000])
def test_route_results_apart(qmlp, rows):
    """the results of the router share no memory: one that is written leaves the others, one that is kept keeps nothing else"""
    r = qmlp.route(rand(20, (rows, 12)), 3)
    assert len({t.untyped_storage().data_ptr() for t in r}) == 5 and all(t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * 4 for t in r)
    kept = [t.clone() for t in r]
    for i, t in enumerate(r):
        t.fill_(-7)
        for other in range(i + 1, 5):
            assert torch.equal(r[other], kept[other])


def test_compiled(qmlp):
    """traced by torch.compile, the operators give what they give without: results and gradients"""
    def model(tokens, table, w, b, router, weight, bias):
        x = qmlp.layer_norm(qmlp.embedding(tokens, table, 2.0), w, b)
        r = qmlp.route(x.float() @ router, 2)
        return qmlp.combine(qmlp.expert_linear(qmlp.dispatch(x, r), weight, r.offsets, bias), r)
    half = torch.float16
    tokens = torch.arange(300, device="cuda") % 41
    leaves = [t.requires_grad_() for t in (rand(30, (40, 16), half), rand(31, (16,)), rand(32, (16,)), rand(33, (16, 6)), rand(34, (6, 24, 16), half), rand(35, (6, 24), half))]
    grad = rand(36, (300, 24), half)
    results = []
    for call in (model, torch.compile(model, fullgraph=True, backend="aot_eager")):
        y = call(tokens, *leaves)
        results.append([y.detach(), *torch.autograd.grad(y, leaves, grad)])
    for a, e in zip(*results):
        assert torch.equal(a, e)


@pytest.mark.parametrize("scale", [float("inf"), float("nan"), -2.0])
def test_embedding_masked_rows(qmlp, scale):
    """masked tokens give rows of zeros and no gradient, whatever the scale"""
    table = rand(40, (20, 24), torch.float16).requires_grad_()
    tokens = torch.tensor([3, -1, 20, 7, 3, 2 ** 40], device="cuda")
    y = qmlp.embedding(tokens, table, scale)
    assert not y[[1, 2, 5]].any() and torch.allclose(y[[0, 3, 4]], table[[3, 7, 3]] * scale, rtol=2.0 ** -11, atol=0, equal_nan=True)
    dt, = torch.autograd.grad(y, table, torch.ones_like(y))
    hit = torch.zeros(20, dtype=torch.bool, device="cuda")
    hit[3] = hit[7] = True
    assert not dt[~hit].any() and (torch.isnan(dt[hit]) | (dt[hit] != 0)).all()
