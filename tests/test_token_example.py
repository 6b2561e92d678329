"""The operators on tokens together with the fused network and activation, as examples/token_experts.py uses them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def example():
    if os.environ.get("QMLP_WARM_CACHE"):
        pytest.skip("nothing to compile ahead that other tests do not")
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_experts.py")
    spec = importlib.util.spec_from_file_location("token_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_experts_match_plain_layers():
    """The layer of experts against every expert applied to all tokens, and its gradients."""
    module = example()
    torch.manual_seed(3)
    layer = module.Experts(5, 24, 40)
    x = torch.randn(70, 24, device="cuda", requires_grad=True)
    grad = torch.randn(70, 24, device="cuda")
    y = layer(x)
    gradients = torch.autograd.grad(y, [x, *layer.parameters()], grad)

    def plain(x):
        normal = torch.nn.functional.layer_norm(x, (24,), layer.norm.weight, layer.norm.bias)
        weights, chosen = torch.softmax(layer.router(normal), 1).topk(2, 1)
        hidden = torch.nn.functional.celu(torch.einsum("nc,ehc->neh", normal, layer.first.weight) + layer.first.bias)
        out = torch.einsum("neh,ech->nec", hidden, layer.second.weight) + layer.second.bias
        return x + (out.gather(1, chosen[..., None].expand(-1, -1, 24)) * weights[..., None]).sum(1)

    expected = plain(x)
    # the experts work in half precision: a handful of roundings of 2^-11 on the way, of values of about one
    torch.testing.assert_close(y, expected, rtol=5e-3, atol=5e-3)
    for a, e in zip(gradients, torch.autograd.grad(expected, [x, *layer.parameters()], grad)):
        torch.testing.assert_close(a, e, rtol=2e-2, atol=2e-2 * float(e.abs().max()))


def test_example_learns():
    losses = example().train(steps=120)
    assert sum(losses[-10:]) < 0.2 * sum(losses[:10])
