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


@pytest.mark.parametrize("which", range(3))
def test_saved_tensors_that_come_back_elsewhere_are_refused(which):
    """No kernel is given an address of the host: neither that of a saved tensor nor that of a gradient given by hand."""
    name, part, arguments = parts()[which]
    print(name, flush=True)
    leaves = [a.detach().requires_grad_() for a in arguments]
    call = {"embedding": lambda t: tokens.embedding(torch.arange(30, device="cuda"), t), "layer norm": tokens.layer_norm,
            "experts": lambda x, w, b: tokens.grouped_linear(x, w, torch.tensor([0, 20, 20, 90], dtype=torch.int32, device="cuda"), b)}[name]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        y = call(*leaves)
    with pytest.raises(RuntimeError, match="another device"):
        y.backward(torch.ones_like(y))
    # one of them alone
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or len(saved) - 1, lambda i: saved[i].cpu() if i == len(saved) - 1 else saved[i]):
        y = call(*leaves)
    with pytest.raises(RuntimeError, match="another device"):
        y.backward(torch.ones_like(y))
    y = call(*leaves)
    with pytest.raises(RuntimeError, match="GPU"):
        y.grad_fn(torch.ones(y.shape))
    # and on the GPU again, they do
    with torch.autograd.graph.save_on_cpu():
        away = call(*leaves)
    for a, e in zip(torch.autograd.grad(away, leaves, torch.ones_like(y)), torch.autograd.grad(y, leaves, torch.ones_like(y))):
        assert torch.equal(a, e)


def test_statistics_in_another_form_are_refused():
    x = torch.randn(70, 40, device="cuda", requires_grad=True)
    for change in (lambda t: t.t().contiguous().t(), lambda t: t[:1], lambda t: t[0]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: change(t) if t.shape == (2, 70) else t):
            y = tokens.layer_norm(x)
        with pytest.raises(RuntimeError, match="another form"):
            y.backward(torch.ones_like(y))
    assert x.grad is None
