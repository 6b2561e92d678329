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


def test_gradients_of_experts_too_large_for_a_launch_are_refused_as_a_whole():
    """1024 matrices of 2^30 entries have 2^26 tiles: refused before the gradient of the input is launched, which alone were small enough."""
    lib, H, I = _lib.lib, _lib.QMLP_HALF, _lib.QMLP_INT32
    rows, weight = descriptor(H, 64, 32768), descriptor(H, 1024, 32768, 32768)
    none = _lib.TensorDesc()
    refused(lib.qmlp_tokens_grouped_linear_adjoint(rows, weight, descriptor(I, 1025), rows, rows, weight, none, 256, None), "too large for one launch")


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


# ------------------------------------------------------------------------------------------------ rare branches
@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("groups", [(1 << 24) - 1, 1 << 24, (1 << 24) + 12345])
def test_groups_of_two_and_three_passes(groups, dtype):
    """2^24 groups and the rows of none have 25 bits: three passes."""
    print("groups", groups, dtype, flush=True)
    rng = np.random.default_rng(groups)
    index = rng.integers(-2, groups + 3, 50001)
    index[::7] = groups - 1
    index[::11] = 4099
    order, offsets = tokens.group(torch.from_numpy(index).to(dtype).cuda(), groups)
    key = np.where((index >= 0) & (index < groups), index, groups)
    assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
    assert np.array_equal(offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(groups + 1)))


@gpu
@pytest.mark.parametrize("channels,dtype", [(5, torch.float32), (64, torch.float16)])
def test_gradient_of_a_token_with_blocks_of_the_third_size(channels, dtype):
    """2^18 places per block: most of 2^20 + 777 rows name one token, which begins in the middle of a block. Whole numbers: sums are exact."""
    rows = (1 << 20) + 777
    g = torch.Generator(device="cuda").manual_seed(70)
    index = torch.full((rows,), 3, device="cuda")
    index[torch.randperm(rows, device="cuda", generator=g)[:5000]] = torch.randint(-1, 9, (5000,), device="cuda", generator=g)
    grad = torch.randint(-2, 3, (rows, channels), device="cuda", generator=g).to(dtype)
    table = torch.zeros(9, channels, dtype=dtype, device="cuda", requires_grad=True)
    dtable, = torch.autograd.grad(tokens.embedding(index, table), table, grad)
    exact = torch.stack([grad[index == v].double().sum(0) for v in range(9)])
    assert torch.equal(dtable, exact.to(dtype))   # (halves: rounded once, below 2^24)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[3000, 0, 1, 2000, 500], [7] * 600], ids=["several chunks", "one chunk each"])
def test_gradient_of_the_biases_alone(counts, dtype):
    """Small whole numbers, sums that every type holds."""
    g = torch.Generator(device="cuda").manual_seed(71)
    experts, rows = len(counts), sum(counts) + 4
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    x, weight = torch.randn(rows, 40, device="cuda", generator=g).to(dtype), torch.randn(experts, 72, 40, device="cuda", generator=g).to(dtype)
    bias = torch.zeros(experts, 72, dtype=dtype, device="cuda", requires_grad=True)
    grad = (torch.rand(rows, 72, device="cuda", generator=g) < 0.03).to(dtype)
    db, = torch.autograd.grad(tokens.grouped_linear(x, weight, offsets, bias), bias, grad)
    expert = torch.repeat_interleave(torch.arange(experts, device="cuda"), torch.tensor(counts, device="cuda"))
    exact = torch.zeros(experts, 72, dtype=torch.float64, device="cuda").index_add_(0, expert, grad[:rows - 4].double())
    assert float(exact.max()) < 256
    assert torch.equal(db.double(), exact)


# ------------------------------------------------------------------------------------------------ memory beside the tensors
class Margins:
    """Tensors inside of one buffer of a known pattern, with 64 KB of it on either side of each."""
    MARGIN, PATTERN = 1 << 16, 0x5A

    def __init__(self, megabytes=64):
        self.buffer = torch.full((megabytes << 20,), self.PATTERN, dtype=torch.uint8, device="cuda")
        self.at, self.used = self.MARGIN, []

    def bytes(self, count):
        """Device address of so many bytes."""
        start = self.at
        self.used.append((start, start + count))
        self.at = -(-(start + count) // 256) * 256 + self.MARGIN
        assert self.at <= self.buffer.numel()
        return self.buffer.data_ptr() + start

    def tensor(self, precision, *sizes, size):
        return descriptor(precision, *sizes, data=self.bytes(int(np.prod(sizes)) * size))

    def untouched(self):
        end = 0
        for start, stop in self.used:
            assert bool((self.buffer[end:start] == self.PATTERN).all()), "before %d" % start
            end = stop
        assert bool((self.buffer[end:] == self.PATTERN).all()), "behind the last"


@gpu
@pytest.mark.parametrize("offsets", [[0, 50, 1 << 30, 1 << 30, 1 << 30], [0, -5, -7, 1000, 20], [90, 80, 70, 60, 50], [2 ** 31 - 1] * 5, [-2 ** 31] * 5,
                                     [0, 33, 33, 64, 97]])
@pytest.mark.parametrize("precision,dtype", [(_lib.QMLP_FLOAT, torch.float32), (_lib.QMLP_BFLOAT16, torch.bfloat16)])
@pytest.mark.parametrize("rows,inputs,outputs", [(97, 16, 24), (97, 2001, 33), (2100, 64, 72)])
def test_nothing_beside_the_results_of_experts_is_written(offsets, precision, dtype, rows, inputs, outputs):
    """Offsets that make no sense give no sensible rows, but what the calls write is within their results and their memory."""
    print("experts beside", offsets, dtype, rows, inputs, outputs, flush=True)
    lib, size = _lib.lib, ctypes.c_size_t()
    margins, es = Margins(), torch.empty(0, dtype=dtype).element_size()
    x, weight, dy = (torch.ones(*s, dtype=dtype, device="cuda") for s in ((rows, inputs), (4, outputs, inputs), (rows, outputs)))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    of = lambda t, p: descriptor(p, *t.shape, data=t.data_ptr())  # noqa: E731
    tx, tw, tdy, to = of(x, precision), of(weight, precision), of(dy, precision), of(off, _lib.QMLP_INT32)
    none, stream = _lib.TensorDesc(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    y, dx = margins.tensor(precision, rows, outputs, size=es), margins.tensor(precision, rows, inputs, size=es)
    dw, db = margins.tensor(precision, 4, outputs, inputs, size=es), margins.tensor(precision, 4, outputs, size=es)
    _lib.check(lib.qmlp_tokens_grouped_linear_memory(rows, 4, inputs, outputs, ctypes.byref(size)))
    memory = margins.bytes(size.value)
    assert memory % 256 == 0
    _lib.check(lib.qmlp_tokens_grouped_linear(tx, tw, to, none, y, memory, stream))
    _lib.check(lib.qmlp_tokens_grouped_linear_adjoint_memory(rows, 4, inputs, outputs, ctypes.byref(size)))
    memory = margins.bytes(size.value)
    _lib.check(lib.qmlp_tokens_grouped_linear_adjoint(tx, tw, to, tdy, dx, dw, db, memory, stream))
    torch.cuda.synchronize()
    margins.untouched()


@gpu
@pytest.mark.parametrize("precision,dtype", [(_lib.QMLP_FLOAT, torch.float32), (_lib.QMLP_HALF, torch.float16)])
@pytest.mark.parametrize("rows,vocabulary,channels", [(1, 1, 1), (300, 7, 9), (9000, 5000, 33), (70001, 40, 17)])
def test_nothing_beside_the_results_of_lookups_and_norms_is_written(precision, dtype, rows, vocabulary, channels):
    print("lookups and norms beside", dtype, rows, vocabulary, channels, flush=True)
    lib, size = _lib.lib, ctypes.c_size_t()
    margins, es = Margins(), torch.empty(0, dtype=dtype).element_size()
    index = torch.arange(rows, dtype=torch.int32, device="cuda") % (vocabulary + 2) - 1
    table, grad = torch.ones(vocabulary, channels, dtype=dtype, device="cuda"), torch.ones(rows, channels, dtype=dtype, device="cuda")
    of = lambda t, p: descriptor(p, *t.shape, data=t.data_ptr())  # noqa: E731
    ti, tt, tg = of(index, _lib.QMLP_INT32), of(table, precision), of(grad, precision)
    none, stream = _lib.TensorDesc(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    I32, F32 = _lib.QMLP_INT32, _lib.QMLP_FLOAT

    def memory(function, *arguments):
        _lib.check(function(*arguments, ctypes.byref(size)))
        return margins.bytes(size.value)

    order, offsets = margins.tensor(I32, rows, size=4), margins.tensor(I32, vocabulary + 1, size=4)
    _lib.check(lib.qmlp_tokens_group(ti, vocabulary, order, offsets, memory(lib.qmlp_tokens_group_memory, rows, vocabulary), stream))
    _lib.check(lib.qmlp_tokens_embedding(ti, tt, 1.0, margins.tensor(precision, rows, channels, size=es), stream))
    adjoint = memory(lib.qmlp_tokens_embedding_adjoint_memory, rows, vocabulary, channels)
    _lib.check(lib.qmlp_tokens_embedding_adjoint(ti, tg, 1.0, margins.tensor(precision, vocabulary, channels, size=es), adjoint, stream))
    mean, rstd = margins.tensor(F32, rows, size=4), margins.tensor(F32, rows, size=4)
    _lib.check(lib.qmlp_tokens_layer_norm(tg, none, none, 1e-5, margins.tensor(precision, rows, channels, size=es), mean, rstd, stream))
    adjoint = memory(lib.qmlp_tokens_layer_norm_adjoint_memory, rows, channels)
    _lib.check(lib.qmlp_tokens_layer_norm_adjoint(tg, none, mean, rstd, tg, margins.tensor(precision, rows, channels, size=es),
                                                  margins.tensor(precision, channels, size=es), margins.tensor(precision, channels, size=es), adjoint, stream))
    torch.cuda.synchronize()
    margins.untouched()
