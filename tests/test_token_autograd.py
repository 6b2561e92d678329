"""The backward passes of the operators on tokens as autograd runs them: with saved tensors that hooks replace or make again."""
import os

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from qmlp import tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_warming():
    if os.environ.get("QMLP_WARM_CACHE"):
        pytest.skip("kernels are compiled by qmlp.tokens.precompile")


def parts():
    """Name, a part of a model that begins with operators of torch and ends with one on tokens, and its arguments."""
    g = torch.Generator(device="cuda").manual_seed(50)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g).requires_grad_()  # noqa: E731
    index = torch.randint(-1, 30, (90,), device="cuda", generator=g)
    offsets = torch.tensor([0, 20, 20, 90], dtype=torch.int32, device="cuda")
    return [("embedding", lambda t: tokens.embedding(index, torch.tanh(t * 2), 1.5), (normal(30, 12),)),
            ("layer norm", lambda x, w, b: tokens.layer_norm(torch.exp(x) * x, w.square(), b), (normal(90, 40), normal(40), normal(40))),
            ("experts", lambda x, w, b: tokens.grouped_linear(torch.sigmoid(x), w.square(), offsets, b), (normal(90, 16), normal(3, 24, 16), normal(3, 24)))]


@pytest.mark.parametrize("which", range(3))
def test_checkpointed_parts_have_the_same_gradients(which):
    """The part is run again when the first saved tensor of its last operator is asked for: with everything recorded that the first run recorded."""
    name, part, arguments = parts()[which]
    print(name, flush=True)
    y = part(*arguments)
    grad = torch.cos(torch.arange(y.numel(), device="cuda", dtype=torch.float32)).view(y.shape)
    expected = torch.autograd.grad(y, arguments, grad)
    again = checkpoint(part, *arguments, use_reentrant=False)
    assert torch.equal(again, y)
    for a, e in zip(torch.autograd.grad(again, arguments, grad), expected):
        assert torch.equal(a, e)
