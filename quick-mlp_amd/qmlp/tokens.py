"""Operators on rows of tokens: what a model of tokens with experts needs beside networks and encodings.

All of them work on GPU tensors of type float32, float16 or bfloat16, run on torch's current stream, hold their sums in
32 bits and round once. They are differentiable (once, in reverse mode) in every floating-point argument, those on numbers of 4 bits
(:class:`Mx4`) excepted; the same inputs give the same bits. They have no counterpart in the reference.
"""
import math

import torch

from . import _lib, _native
from ._lib import check, lib

_PRECISION_OF = {torch.float32: _lib.QMLP_FLOAT, torch.float16: _lib.QMLP_HALF, torch.bfloat16: _lib.QMLP_BFLOAT16}


def group(index: torch.Tensor, groups: int, places: bool = False):
    """
    Rows in the order of the group that they belong to, in their own order within a group.

    :param index: (rows) int32 or int64, the group of a row; rows whose index is not in 0 .. groups - 1 belong to none
    :param groups: number of groups
    :param places: whether the place of every row in the order is returned, too
    :return: ``(order, offsets)``, both int32: ``order[offsets[g]:offsets[g + 1]]`` are the rows of group g;
        ``order[offsets[groups]:]`` those of no group. With places ``(order, offsets, places)``: places, int32 of the shape of index,
        for :func:`dispatch` and :func:`combine`; -1 - place for the rows of no group
    """
    return _native.group(index, groups, places)


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


def route(logits: torch.Tensor, chosen: int, normalised: bool = False):
    """
    The router's choice: for every row of logits the experts with the largest ones, the first of equals, in that order, and their shares of the
    softmax. Differentiable in the logits.

    No row takes an expert whose logit is -inf: where a row has fewer others than are chosen, -1 and a weight of 0 stand for the rest. A NaN counts
    as the largest logit; weights of a row with a NaN or +inf are NaN.

    :param logits: (..., experts)
    :param chosen: experts of a row, 1 to 64
    :param normalised: softmax over the chosen experts alone, so that the weights of a row add up to 1
    :return: ``(weights, index)``, both (..., chosen): weights of the logits' type, index int32, for :func:`group`
    """
    return _native.route(logits, chosen, normalised)


def dispatch(x: torch.Tensor, places: torch.Tensor) -> torch.Tensor:
    """
    Rows of tokens to their experts: ``rows[places[..., j]] = x[...]``, zeros at places of no expert. Differentiable in x.

    :param x: (..., channels)
    :param places: (..., chosen) int32, as :func:`group` returns them for the chosen experts: those of a permutation (what any others than that
        leave in the rows is undefined, though nothing beside them is written)
    :return: (tokens * chosen, channels), rows by expert, for :func:`grouped_linear` and :func:`mx4_linear`
    """
    return _native.dispatch(x, places)


def combine(rows: torch.Tensor, places: torch.Tensor, weights: torch.Tensor = None, residual: torch.Tensor = None) -> torch.Tensor:
    """
    And back: ``residual[...] + sum over j of weights[..., j] * rows[places[..., j]]``, without the terms of no expert. Differentiable in rows,
    weights and residual; for the backward pass rows are kept where weights want a gradient, weights where rows do.

    :param rows: (tokens * chosen, channels)
    :param places: (..., chosen) as for :func:`dispatch`
    :param weights: (..., chosen), of the type of the rows or float32; None: 1
    :param residual: (..., channels), of the type of the rows; None: 0
    :return: (..., channels)
    """
    return _native.combine(rows, places, weights, residual)


class Mx4:
    """
    A tensor of 4-bit numbers, blocks of 32 consecutive entries of its last dimension with a common power of two: MXFP4 as the OCP Microscaling
    Formats specification 1.0 has it.

    :param codes: (..., 16 * blocks) uint8, two numbers a byte, the first in the low bits: sign, two bits of exponent, one of mantissa. Zeros
        behind the last column
    :param scales: (..., blocks) uint8, the exponents of the blocks plus 127; 255: a block of NaN
    :param columns: entries of the last dimension, in ceil(columns / 32) blocks
    """
    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int):
        if scales.shape[-1] != (columns + 31) // 32 or codes.shape[-1] != 16 * scales.shape[-1]:
            raise ValueError("%d columns are %d blocks of 16 bytes of codes and a scale, but there are %d bytes and %d scales"
                             % (columns, (columns + 31) // 32, codes.shape[-1], scales.shape[-1]))
        self.codes, self.scales, self.columns = codes, scales, columns

    @property
    def shape(self):
        return torch.Size((*self.scales.shape[:-1], self.columns))

    def dequantise(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the numbers stand for, rounded once to the type (float32 and bfloat16 hold all of them)."""
        return _native.mx4_values(self.codes, self.scales, self.columns, dtype)

    def __repr__(self):
        return "Mx4(%s)" % (tuple(self.shape),)


def quantise_mx4(x: torch.Tensor) -> Mx4:
    """
    x in numbers of 4 bits. The scale of a block is the power of two that brings its largest magnitude to 4 .. 8; its entries go to the nearest of 0,
    0.5, 1, 1.5, 2, 3, 4, 6 times the scale, halfway to the even code. A block with an infinity or a NaN becomes NaN. No gradient: inputs that want
    one are refused.

    :param x: (..., columns)
    """
    return Mx4(*_native.mx4_quantise(x), x.shape[-1])


def mx4_linear(x, weight: Mx4, offsets: torch.Tensor = None, bias: torch.Tensor = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """
    :func:`grouped_linear` with weights of 4 bits, for serving: both operands of the product are numbers of 4 bits, sums are held in 32. No gradient:
    inputs that want one are refused.

    :param x: (rows, inputs), which the call quantises as :func:`quantise_mx4` does, or :class:`Mx4`
    :param weight: (experts, outputs, inputs), quantised along the inputs
    :param offsets: as for :func:`grouped_linear`; None: one expert has all rows
    :param bias: (experts, outputs) of the type of the result, or None
    :param dtype: of the result, where x is :class:`Mx4`; otherwise it has the type of x
    :return: (rows, outputs)
    """
    values, scales, inputs = (x.codes, x.scales, x.columns) if isinstance(x, Mx4) else (x, None, x.shape[-1])
    if inputs != weight.columns:
        raise ValueError("x has rows of %d, the weights of %d inputs" % (inputs, weight.columns))
    return _native.mx4_linear(values, scales, weight.codes, weight.scales, offsets, bias, dtype)


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


class FusedMx4GroupedLinear(torch.nn.Module):
    """The layers of a :class:`FusedGroupedLinear` with weights of 4 bits, for serving: :func:`mx4_linear` with them. Made once from the trained
    layer; codes and scales are buffers."""

    def __init__(self, layer: FusedGroupedLinear):
        super().__init__()
        weight = quantise_mx4(layer.weight.detach())
        self.inputs = weight.columns
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", layer.bias.detach().clone() if layer.bias is not None else None)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        bias = self.bias.to(x.dtype) if self.bias is not None else None
        return mx4_linear(x, Mx4(self.codes, self.scales, self.inputs), offsets, bias)

    def extra_repr(self):
        experts, outputs = self.scales.shape[:2]
        return "%d experts, %d -> %d, bias=%s" % (experts, self.inputs, outputs, self.bias is not None)
