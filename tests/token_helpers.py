"""What the tests of the operators around experts have in common."""
import os

import numpy as np
import pytest
import torch

from qmlp import _lib

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUNDING = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half of the distance of the smallest numbers
U = 2.0 ** -23


def skip_warming(request):
    """(a pass without a GPU that fills the kernel cache: these kernels do not depend on the test)"""
    if os.environ.get("QMLP_WARM_CACHE") and "gpu" in request.keywords:
        pytest.skip("kernels are compiled by qmlp.tokens.precompile")


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def near(value, exact, error, what):
    """value: as computed; error: how far its 32-bit value may be from the exact one, before it is rounded to its type."""
    assert value.shape == exact.shape, what
    assert torch.equal(value.isnan(), exact.isnan()), what
    bound = error + ROUNDING[value.dtype] * (exact.abs() + error) + SMALLEST[value.dtype]
    off = torch.where(exact.isnan(), 0.0, (value.double() - exact).abs())
    assert bool((off <= torch.where(exact.isnan(), 0.0, bound)).all()), "%s: %g of the bound" % (what, float((off / bound.clamp_min(1e-300)).max()))


def say(*what):
    print(*what, flush=True)


def offsets_of(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def descriptor(precision, *sizes, strides=None, data=256):
    d = _lib.TensorDesc()
    d.data, d.precision, d.ndim = data, precision, len(sizes)
    for i, s in enumerate(sizes):
        d.sizes[i] = s
        d.strides[i] = strides[i] if strides else int(np.prod(sizes[i + 1:]))
    return d


def described(t):
    precision = {torch.float32: _lib.QMLP_FLOAT, torch.float16: _lib.QMLP_HALF, torch.bfloat16: _lib.QMLP_BFLOAT16, torch.int32: _lib.QMLP_INT32,
                 torch.uint8: _lib.QMLP_UINT8}[t.dtype]
    return descriptor(precision, *t.shape, strides=t.stride(), data=t.data_ptr())


def refused(rc, match):
    message = _lib.lib.qmlp_last_error().decode()
    assert rc == 2 and match in message, (rc, message)


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

    def tensor(self, dtype, *sizes):
        count = int(np.prod(sizes)) * torch.empty(0, dtype=dtype).element_size()
        start = self.bytes(count) - self.buffer.data_ptr()
        return self.buffer[start:start + count].view(dtype).view(sizes)

    def untouched(self):
        end = 0
        for start, stop in self.used:
            assert bool((self.buffer[end:start] == self.PATTERN).all()), "before %d" % start
            end = stop
        assert bool((self.buffer[end:] == self.PATTERN).all()), "behind the last"
