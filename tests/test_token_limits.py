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
