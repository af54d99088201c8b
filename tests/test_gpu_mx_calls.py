"""4-bit layers as a program calls them: cast as a whole."""
import pytest
import torch

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
