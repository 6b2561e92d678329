"""Operators on rows of tokens: what a model of tokens with experts needs beside networks and encodings.

All of them work on GPU tensors of type float32, float16 or bfloat16, run on torch's current stream, hold their sums in
32 bits and round once. They are differentiable (once, in reverse mode) in every floating-point argument; the same inputs give
the same bits. They have no counterpart in the reference.
"""
import math

import torch

from . import _lib, _native
from ._lib import check, lib

_PRECISION_OF = {torch.float32: _lib.QMLP_FLOAT, torch.float16: _lib.QMLP_HALF, torch.bfloat16: _lib.QMLP_BFLOAT16}


def group(index: torch.Tensor, groups: int):
    """
    Rows in the order of the group that they belong to, in their own order within a group.

    :param index: (rows) int32 or int64, the group of a row; rows whose index is not in 0 .. groups - 1 belong to none
    :param groups: number of groups
    :return: ``(order, offsets)``, both int32: ``order[offsets[g]:offsets[g + 1]]`` are the rows of group g;
        ``order[offsets[groups]:]`` those of no group
    """
    return _native.group(index, groups)


def embedding(index: torch.Tensor, table: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """
    ``scale * table[index]``; rows of zeros where the index names no row of the table (padding, for instance -1), which
    have no part in the gradient either. The gradient of the table is dense.

    :param index: int32 or int64, any shape
    :param table: (vocabulary, channels)
    :return: the shape of index, and channels
    """
    return _native.embedding(index, table, scale)


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """
    ``(x - mean) / sqrt(variance + eps) * weight + bias``, mean and variance over the last dimension.

    :param weight, bias: (channels), of the type of x or float32, both of one type; None: 1 and 0
    """
    return _native.layer_norm(x, weight, bias, eps)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: torch.Tensor = None) -> torch.Tensor:
    """
    The linear layer of every expert on its own rows: ``x[r] @ weight[e].T + bias[e]`` for the rows r from ``offsets[e]`` to
    ``offsets[e + 1] - 1``; zeros for the rows from ``offsets[experts]`` on.

    :param x: (rows, inputs)
    :param weight: (experts, outputs, inputs), of the type of x
    :param offsets: (experts + 1) int32 on the GPU, from 0 on and not decreasing, as :func:`group` returns them
    :param bias: (experts, outputs) or None
    :return: (rows, outputs)
    """
    return _native.grouped_linear(x, weight, offsets, bias)


def precompile(dtype: torch.dtype = torch.float32) -> None:
    """Compiles the kernels for values of one dtype into the kernel cache; needs no GPU."""
    check(lib.qmlp_tokens_precompile(_PRECISION_OF[dtype]))


class FusedEmbedding(torch.nn.Module):
    """A learned table with one row per token, and :func:`embedding` of it."""

    def __init__(self, vocabulary: int, channels: int, scale: float = 1.0, dtype=torch.float32, device="cuda"):
        super().__init__()
        self.scale = scale
        self.table = torch.nn.Parameter(torch.randn(vocabulary, channels, device=device).to(dtype))

    def forward(self, index: torch.Tensor) -> torch.Tensor:
        return embedding(index, self.table, self.scale)

    def extra_repr(self):
        return "%d, %d, scale=%g" % (*self.table.shape, self.scale)


class FusedLayerNorm(torch.nn.Module):
    """:func:`layer_norm` with a learned weight and bias."""

    def __init__(self, channels: int, eps: float = 1e-5, dtype=torch.float32, device="cuda"):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(channels, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%d, eps=%g" % (self.weight.shape[0], self.eps)


class FusedGroupedLinear(torch.nn.Module):
    """A linear layer per expert, and :func:`grouped_linear` with them, in the type of the rows: as with :class:`qmlp.FusedNetwork` the
    parameters may be float32 for the optimizer while the layers are evaluated in 16 bits."""

    def __init__(self, experts: int, inputs: int, outputs: int, bias: bool = True, dtype=torch.float32, device="cuda"):
        super().__init__()
        bound = 1 / math.sqrt(inputs)
        self.weight = torch.nn.Parameter(torch.empty(experts, outputs, inputs, device=device).uniform_(-bound, bound).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(experts, outputs, dtype=dtype, device=device)) if bias else None

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        bias = self.bias.to(x.dtype) if self.bias is not None else None
        return grouped_linear(x, self.weight.to(x.dtype), offsets, bias)

    def extra_repr(self):
        experts, outputs, inputs = self.weight.shape
        return "%d experts, %d -> %d, bias=%s" % (experts, inputs, outputs, self.bias is not None)
