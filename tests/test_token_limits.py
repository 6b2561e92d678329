"""Sizes of the operators on tokens that are near the ends of what their kernels can count; memory beside their tensors; rare branches."""
import ctypes
import os

import numpy as np
import pytest
import torch

from qmlp import _lib, tokens

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_warming(request):
    if os.environ.get("QMLP_WARM_CACHE") and "gpu" in request.keywords:
        pytest.skip("kernels are compiled by qmlp.tokens.precompile")


def descriptor(precision, *sizes, strides=None, data=256):
    d = _lib.TensorDesc()
    d.data, d.precision, d.ndim = data, precision, len(sizes)
    for i, s in enumerate(sizes):
        d.sizes[i] = s
        d.strides[i] = strides[i] if strides else int(np.prod(sizes[i + 1:]))
    return d


def refused(rc, match):
    message = _lib.lib.qmlp_last_error().decode()
    assert rc == 2 and match in message, (rc, message)


MOST = 2 ** 31 - 2 ** 12


@pytest.mark.parametrize("size", [MOST + 1, 2 ** 31 - 1])
def test_sizes_whose_last_step_has_no_number_are_refused(size):
    """(needs no device: what is refused is never launched)"""
    lib, H, F, I = _lib.lib, _lib.QMLP_HALF, _lib.QMLP_FLOAT, _lib.QMLP_INT32
    none = _lib.TensorDesc()
    row, index = descriptor(H, 1, size), descriptor(I, 1)
    refused(lib.qmlp_tokens_embedding(index, descriptor(H, 1, size), 1.0, row, None), "channels must not be more")
    refused(lib.qmlp_tokens_embedding_adjoint(index, row, 1.0, descriptor(H, 1, size), 256, None), "channels must not be more")
    refused(lib.qmlp_tokens_layer_norm(row, none, none, 1e-5, row, none, none, None), "channels must not be more")
    one = descriptor(F, 1)
    refused(lib.qmlp_tokens_layer_norm_adjoint(row, none, one, one, row, row, none, none, 256, None), "channels must not be more")
    offsets, few = descriptor(I, 2), descriptor(H, 1, 1)
    refused(lib.qmlp_tokens_grouped_linear(row, descriptor(H, 1, 1, size), offsets, none, few, 256, None), "inputs must not be more")
    refused(lib.qmlp_tokens_grouped_linear(few, descriptor(H, 1, size, 1), offsets, none, row, 256, None), "outputs must not be more")
    many = descriptor(H, size, 1)
    for weight in (descriptor(H, 1, 1, 1), none):
        refused(lib.qmlp_tokens_grouped_linear_adjoint(many, descriptor(H, 1, 1, 1), offsets, many, none, weight, few, 256, None), "rows must not be more")


def test_a_gradient_of_too_many_rows_for_a_launch_is_refused():
    """2^31 - 1 rows (all the same one in memory) of more than 512 floats: 2^25 blocks of 64 places, 128 lanes or more for each."""
    lib, F, I = _lib.lib, _lib.QMLP_FLOAT, _lib.QMLP_INT32
    rows = 2 ** 31 - 1
    refused(lib.qmlp_tokens_embedding_adjoint(descriptor(I, rows), descriptor(F, rows, 600, strides=(0, 1)), 1.0, descriptor(F, 4, 600), 256, None),
            "too large for one launch")


@gpu
def test_gradient_of_a_table_of_more_than_two_to_the_30_rows():
    vocabulary = (1 << 30) + 5
    table = torch.zeros(vocabulary, 1, dtype=torch.float16, device="cuda", requires_grad=True)
    index = torch.tensor([vocabulary - 1, 3, vocabulary, 1 << 29, 3, -1, vocabulary - 2], device="cuda")
    y = tokens.embedding(index, table)
    dtable, = torch.autograd.grad(y, table, torch.arange(1, 8, device="cuda").half()[:, None])
    assert [float(dtable[v]) for v in (vocabulary - 1, 3, 1 << 29, vocabulary - 2)] == [1, 7, 4, 7]
    assert int(torch.count_nonzero(dtable)) == 4


@gpu
def test_layer_norm_of_more_columns_than_a_launch_takes_in_one_go():
    """2^26 columns: their sums over the rows have 2^32 threads' work. One row, so that the gradient of the bias is that of the output."""
    channels = (1 << 26) + 7
    g = torch.Generator(device="cuda").manual_seed(60)
    x, grad = (torch.randn(1, channels, device="cuda", generator=g) for _ in range(2))
    weight, bias = (torch.full((channels,), v, device="cuda", requires_grad=True) for v in (1.0, 0.0))
    y = tokens.layer_norm(x, weight, bias)
    dw, db = torch.autograd.grad(y, (weight, bias), grad)
    assert torch.equal(db, grad[0])
    # y is the normal here: the same products, rounded once
    torch.testing.assert_close(dw, (grad * y.detach())[0], rtol=2.0 ** -20, atol=0)


@gpu
def test_layer_norm_of_rows_whose_slices_have_too_many_sums():
    """256 slices of 2^24 columns: 2^32 threads. 257 rows that are all the same in memory, entries of 1 and -1."""
    channels, rows = (1 << 24) + 2, 257
    row = 1 - 2 * (torch.arange(channels, device="cuda") % 2).half()
    weight, bias = (torch.full((channels,), v, dtype=torch.float16, device="cuda", requires_grad=True) for v in (1.0, 0.0))
    y = tokens.layer_norm(row.expand(rows, channels), weight, bias, 0.0)
    dw, db = torch.autograd.grad(y, (weight, bias), torch.ones(1, channels, dtype=torch.float16, device="cuda").expand(rows, channels))
    # (mean 0 and variance 1 are exact, and so are sums up to 257)
    assert torch.equal(db, torch.full_like(db, 257))
    assert torch.equal(dw, 257 * row)
