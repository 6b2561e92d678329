"""Operators on rows of tokens (qmlp.tokens) against their definitions in 64 bits.

Tolerances follow from the operators: sums of n terms are held in 32 bits, which is off by at most n 2^-23 of the sum of their
magnitudes (in any order, with a bit to spare for the matrix cores' own rounding), and a result is rounded once to its type.
"""
import ctypes
import os

import numpy as np
import pytest
import torch

import qmlp
from qmlp import _lib
from qmlp import tokens

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_warming(request):
    """(a pass without a GPU that fills the kernel cache: these kernels do not depend on the test)"""
    if os.environ.get("QMLP_WARM_CACHE") and "gpu" in request.keywords:
        pytest.skip("kernels are compiled by qmlp.tokens.precompile")

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUNDING = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half of the distance of the smallest numbers
U = 2.0 ** -23


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def near(value, exact, error, what):
    """value: as computed; error: how far its 32-bit value may be from the exact one, before it is rounded to its type."""
    assert value.shape == exact.shape, what
    bound = error + ROUNDING[value.dtype] * (exact.abs() + error) + SMALLEST[value.dtype]
    off = (value.double() - exact).abs()
    assert bool((off <= bound).all()), "%s: %g of the bound" % (what, float((off / bound.clamp_min(1e-300)).max()))


def say(*what):
    print(*what, flush=True)


# ------------------------------------------------------------------------------------------------ groups
@gpu
@pytest.mark.parametrize("groups", [0, 1, 2, 8, 255, 256, 4096, 4399, 4400, 8191, 9000, 70000])
@pytest.mark.parametrize("rows", [0, 1, 63, 64, 65, 1000, 8192, 8193, 70001, 300007])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_groups_are_a_stable_sort(rows, groups, dtype):
    say("group", rows, groups, dtype)
    rng = np.random.default_rng(rows + groups)
    index = rng.integers(-2, groups + 3, rows)   # some of no group on either side
    if groups > 3 and rows > 100:
        index[rng.random(rows) < 0.4] = 3        # and a crowded one
    order, offsets = tokens.group(torch.from_numpy(index).to(dtype).cuda(), groups)
    key = np.where((index >= 0) & (index < groups), index, groups)
    assert order.dtype == offsets.dtype == torch.int32
    assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
    assert np.array_equal(offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(groups + 1)))


@gpu
def test_groups_of_strided_and_wide_indices():
    """Every second index of a longer array; 64-bit indices whose lower halves would name a group."""
    index = torch.arange(2 * 20000, device="cuda") % 14
    order, offsets = tokens.group(index[::2], 7)
    key = (2 * np.arange(20000)) % 14
    key[key >= 7] = 7
    assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
    assert offsets.cpu().tolist() == np.searchsorted(np.sort(key), np.arange(8)).tolist()
    wide = torch.tensor([1 << 32, 0, (1 << 40) + 1, -(1 << 32), 1], device="cuda")
    order, offsets = tokens.group(wide, 2)
    assert order.tolist() == [1, 4, 0, 2, 3] and offsets.tolist() == [0, 1, 2]


# ------------------------------------------------------------------------------------------------ embedding
def embedding_reference(index, table, scale, grad):
    index = index.reshape(-1).long()
    valid = (index >= 0) & (index < table.shape[0])
    y = torch.zeros((index.numel(), table.shape[1]), dtype=torch.float64, device=table.device)
    y[valid] = table.double()[index[valid]] * scale
    grad = grad.double().reshape(-1, table.shape[1])
    dtable, size = (torch.zeros(table.shape, dtype=torch.float64, device=table.device) for _ in range(2))
    dtable.index_add_(0, index[valid], grad[valid] * scale)
    size.index_add_(0, index[valid], grad[valid].abs() * abs(scale))
    counts = torch.bincount(index[valid], minlength=table.shape[0]).double()[:, None]
    return y, dtable, (counts + 4) * U * size


@gpu
@pytest.mark.parametrize("rows,vocabulary", [(0, 5), (1, 1), (5, 40), (64, 3), (1000, 1000), (9001, 300), (40000, 20011)])
@pytest.mark.parametrize("channels", [1, 3, 8, 31, 100, 777])
@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_and_its_gradient(rows, vocabulary, channels, dtype):
    say("embedding", rows, vocabulary, channels, dtype)
    g = generator(rows + channels)
    index = torch.randint(-1, vocabulary + 1, (rows,), device="cuda", generator=g)
    if rows >= 1000:   # one token more often than a block of blocks of the sorted order holds
        index[torch.rand(rows, device="cuda", generator=g) < 0.3] = 2
    table, grad = normal(g, vocabulary, channels, dtype=dtype).requires_grad_(), normal(g, rows, channels, dtype=dtype)
    y = tokens.embedding(index.to(torch.int32 if channels % 2 else torch.int64), table, 1.5)
    dtable, = torch.autograd.grad(y, table, grad)
    exact, dexact, error = embedding_reference(index, table.detach(), 1.5, grad)
    near(y.detach(), exact, U * exact.abs(), "rows")
    near(dtable, dexact, error, "gradient")
    again, = torch.autograd.grad(tokens.embedding(index, table, 1.5), table, grad)
    assert torch.equal(dtable, again)


@gpu
@pytest.mark.parametrize("count", [31, 32, 33, 1024, 1025, 40000])
def test_gradient_of_one_token_alone(count):
    g = generator(count)
    index = torch.full((count,), 1, device="cuda")
    index[:3] = 0
    table, grad = normal(g, 4, 40).requires_grad_(), normal(g, count, 40)
    dtable, = torch.autograd.grad(tokens.embedding(index, table), table, grad)
    _, exact, error = embedding_reference(index, table.detach(), 1.0, grad)
    near(dtable, exact, error, "gradient")
    assert torch.equal(dtable[2:], torch.zeros_like(dtable[2:]))


@gpu
def test_embedding_of_other_shapes_and_strides():
    g = generator(1)
    index = torch.randint(0, 50, (6, 7), device="cuda", generator=g).t()
    wide = normal(g, 50, 40)
    for table in (wide[:, 3:20], wide[::2][:, :9], wide.t()[:30], wide[:1].expand(50, 40)):
        table = table.detach().requires_grad_()
        y = tokens.embedding(index, table, -2.0)
        assert y.shape == (7, 6, table.shape[1])
        assert torch.equal(y, -2.0 * table[index.clamp(max=table.shape[0])] if table.shape[0] >= 50 else
                           torch.where((index < table.shape[0])[..., None], -2.0 * table[index.clamp(max=table.shape[0] - 1)], 0.0))
        dtable, = torch.autograd.grad(y.sum(), table)   # (a gradient of the output that is one number in memory)
        counts = torch.bincount(index.reshape(-1), minlength=50)[:table.shape[0]].float()
        assert torch.equal(dtable, (-2.0 * counts)[:, None].expand(table.shape))


@gpu
def test_what_is_not_a_number_stays_in_its_row():
    g = generator(2)
    index = torch.randint(0, 30, (3000,), device="cuda", generator=g)
    table, grad = normal(g, 30, 20).requires_grad_(), normal(g, 3000, 20)
    grad[index == 4] = float("nan")
    grad[(index == 5).nonzero()[0], 7] = float("inf")
    y = tokens.embedding(index, table)
    dtable, = torch.autograd.grad(y, table, grad)
    assert bool(dtable[4].isnan().all()) and float(dtable[5, 7]) == float("inf")
    dtable[4], dtable[5, 7] = 0, 0
    assert bool(dtable.isfinite().all())
    assert torch.equal(tokens.embedding(torch.tensor([-1, 30, -(1 << 40), 1 << 40], device="cuda"), torch.full((30, 20), float("nan"), device="cuda")),
                       torch.zeros(4, 20, device="cuda"))


@gpu
def test_table_of_more_than_two_to_the_31_entries():
    """Rows whose first entries have no 32-bit offset, read and in the gradient."""
    vocabulary, channels = (1 << 31) // 1024 + 5, 1024
    table = torch.zeros(vocabulary, channels, dtype=torch.float16, device="cuda")
    table[-1] = 2
    table.requires_grad_()
    index = torch.tensor([vocabulary - 1, 0, vocabulary - 1], device="cuda")
    y = tokens.embedding(index, table, 0.5)
    assert torch.equal(y, torch.tensor([1.0, 0, 1], device="cuda").half()[:, None].expand(3, channels))
    dtable, = torch.autograd.grad(y, table, torch.ones_like(y))
    assert bool((dtable[-1] == 1).all()) and bool((dtable[0] == 0.5).all())
    assert int(torch.count_nonzero(dtable)) == 2 * channels


# ------------------------------------------------------------------------------------------------ layer norm
def layer_norm_reference(x, weight, bias, eps, grad):
    """Results and how far 32-bit arithmetic may be off them."""
    x, grad = x.double(), grad.double()
    n = x.shape[1]
    w = weight.double() if weight is not None else torch.ones(n, dtype=torch.float64, device=x.device)
    b = bias.double() if bias is not None else torch.zeros(n, dtype=torch.float64, device=x.device)
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    normal_ = d * r
    e_mean = (n + 2) * U * x.abs().mean(1, keepdim=True)
    e_r = 0.5 * ((n + 4) * U + e_mean ** 2 * r * r) + 2 * U        # relative
    e_n = r * (e_mean + U * d.abs()) + normal_.abs() * e_r + U * normal_.abs()
    y = normal_ * w + b
    e_y = w.abs() * e_n + 2 * U * ((normal_ * w).abs() + b.abs())
    h = grad * w
    a, c = h.mean(1, keepdim=True), (h * normal_).mean(1, keepdim=True)
    e_a = (n + 4) * U * h.abs().mean(1, keepdim=True)
    e_c = (h.abs() * e_n).mean(1, keepdim=True) + (n + 4) * U * (h * normal_).abs().mean(1, keepdim=True)
    dx = r * (h - a - normal_ * c)
    e_dx = r * (e_a + e_n * c.abs() + normal_.abs() * e_c + e_n * e_c + 4 * U * (h.abs() + a.abs() + (normal_ * c).abs())) * (1 + e_r) + e_r * dx.abs()
    rows = x.shape[0]
    e_dw = (grad.abs() * e_n).sum(0) + (rows + 4) * U * (grad * normal_).abs().sum(0)
    e_db = (rows + 4) * U * grad.abs().sum(0)
    return (y, e_y), (dx, e_dx), ((grad * normal_).sum(0), e_dw), (grad.sum(0), e_db)


@gpu
@pytest.mark.parametrize("channels", [1, 2, 7, 8, 9, 64, 65, 130, 333, 777, 1024, 1500, 4096, 5001, 12000, 20000, 33000])
@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_and_its_gradients(rows, channels, dtype):
    say("layer norm", rows, channels, dtype)
    g = generator(channels + rows)
    x = (3 * normal(g, rows, channels) + normal(g, channels)).to(dtype).requires_grad_()
    weight, bias = ((1 + 0.3 * normal(g, channels)).to(dtype).requires_grad_(), normal(g, channels).to(dtype).requires_grad_())
    grad = normal(g, rows, channels, dtype=dtype)
    y = tokens.layer_norm(x, weight, bias, 1e-3)
    gradients = torch.autograd.grad(y, (x, weight, bias), grad)
    exact = layer_norm_reference(x.detach(), weight.detach(), bias.detach(), 1e-3, grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight", "bias")):
        near(value, expected, error, what)
    with torch.no_grad():
        assert torch.equal(tokens.layer_norm(x, weight, bias, 1e-3), y)
    for a, b in zip(gradients, torch.autograd.grad(tokens.layer_norm(x, weight, bias, 1e-3), (x, weight, bias), grad)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("affine", ["float weights", "no weight", "no bias", "nothing"])
def test_layer_norm_with_other_weights(dtype, affine):
    g = generator(5)
    x = normal(g, 50, 300, dtype=dtype).requires_grad_()
    weight = None if affine in ("no weight", "nothing") else (1 + normal(g, 300)).requires_grad_()
    bias = None if affine in ("no bias", "nothing") else normal(g, 300).requires_grad_()
    grad = normal(g, 50, 300, dtype=dtype)
    y = tokens.layer_norm(x, weight, bias)
    wanted = [t for t in (x, weight, bias) if t is not None]
    exact = layer_norm_reference(x.detach(), weight, bias, 1e-5, grad)
    near(y.detach(), *exact[0], "y")
    gradients = torch.autograd.grad(y, wanted, grad)
    expected = [e for e, t in zip(exact[1:], (x, weight, bias)) if t is not None]
    for t, value, (e, error) in zip(wanted, gradients, expected):
        assert value.dtype == t.dtype
        near(value, e.detach(), error.detach(), "gradient")


@gpu
def test_layer_norm_takes_any_shape_and_stride():
    g = generator(6)
    wide = normal(g, 40, 3, 70)
    weight, bias = normal(g, 200)[::4][:50], normal(g, 50)
    for x in (wide[..., 5:55], wide[::3, :, 20:], wide.transpose(0, 2)[:, :, :1].expand(70, 3, 50), wide.permute(1, 2, 0)[..., :50].repeat(1, 1, 2)[..., :50]):
        x = x.detach().requires_grad_()
        y = tokens.layer_norm(x, weight, bias)
        dx, = torch.autograd.grad(y.sum(), x)
        flat = x.detach().reshape(-1, 50)
        (ey, ery), (edx, erdx), _, _ = layer_norm_reference(flat, weight, bias, 1e-5, torch.ones_like(flat))
        assert y.shape == dx.shape == x.shape
        near(y.detach().reshape(-1, 50), ey, ery, "y")
        near(dx.reshape(-1, 50), edx, erdx, "x")
    empty = torch.empty(0, 50, device="cuda", requires_grad=True)
    w = weight.clone().requires_grad_()
    dx, dw = torch.autograd.grad(tokens.layer_norm(empty, w, bias).sum(), (empty, w))
    assert dx.shape == (0, 50) and torch.equal(dw, torch.zeros(50, device="cuda"))


@gpu
@pytest.mark.parametrize("channels", [40, 3000, 33000])
def test_rows_of_a_layer_norm_do_not_mix(channels):
    """Infinities and NaN stay in their rows; a row of equal values has no variance; a large mean costs no digits of the rest."""
    g = generator(7)
    x = normal(g, 9, channels)
    x[2, 3], x[5, 1] = float("inf"), float("nan")
    x[7] = 4.0
    x[8] = 1000 + x[8]
    x.requires_grad_()
    y = tokens.layer_norm(x)
    dx, = torch.autograd.grad(y, x, normal(g, 9, channels))
    for r in (2, 5):
        assert bool(y[r].isnan().all()) and bool(dx[r].isnan().all())
    keep = [0, 1, 3, 4, 6, 7, 8]
    assert bool(y[keep].isfinite().all()) and bool(dx[keep].isfinite().all())
    assert torch.equal(y[7], torch.zeros_like(y[7]))
    (ey, ery), _, _, _ = layer_norm_reference(x.detach()[8:], None, None, 1e-5, x.detach()[8:])
    near(y.detach()[8:], ey, ery, "large mean")


# ------------------------------------------------------------------------------------------------ grouped linear layers
def offsets_of(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")


def grouped_reference(x, weight, counts, bias, grad):
    x, weight, grad = x.double(), weight.double(), grad.double()
    experts, outputs, inputs = weight.shape
    y, ey = (torch.zeros(x.shape[0], outputs, dtype=torch.float64, device=x.device) for _ in range(2))
    dx, edx = torch.zeros_like(x), torch.zeros_like(x)
    dw, edw = torch.zeros_like(weight), torch.zeros_like(weight)
    db, edb = (torch.zeros(experts, outputs, dtype=torch.float64, device=x.device) for _ in range(2))
    at = 0
    for e, n in enumerate(counts):
        p = slice(at, at + n)
        at += n
        y[p] = x[p] @ weight[e].T + (bias[e].double() if bias is not None else 0)
        ey[p] = (inputs + 8) * U * (x[p].abs() @ weight[e].abs().T + (bias[e].double().abs() if bias is not None else 0))
        dx[p], edx[p] = grad[p] @ weight[e], (outputs + 8) * U * (grad[p].abs() @ weight[e].abs())
        dw[e], edw[e] = grad[p].T @ x[p], (n + 8) * U * (grad[p].abs().T @ x[p].abs())
        db[e], edb[e] = grad[p].sum(0), (n + 8) * U * grad[p].abs().sum(0)
    return (y, ey), (dx, edx), (dw, edw), (db, edb)


COUNTS = {
    "one row": [1],
    "one row of many experts": [0, 0, 1, 0] + [0] * 70,
    "nothing": [0, 0, 0],
    "ragged": [5, 0, 130, 1, 64, 0, 0, 257, 33],
    "one has all": [0, 0, 3000, 0],
    "hundreds of experts": [(7 * i) % 13 for i in range(300)],
    "many rows": [5000, 4097, 1],
}


@gpu
@pytest.mark.parametrize("inputs,outputs", [(2000, 40), (40, 2000), (1023, 1100)])
@pytest.mark.parametrize("counts", [[1], [3, 0, 9], [70, 0, 0, 31]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums_of_few_rows(inputs, outputs, counts, dtype):
    """Sums that are shared out over workgroups and joined."""
    say("long sums", inputs, outputs, counts, dtype)
    g = generator(inputs)
    rows = sum(counts) + 2
    x, weight = normal(g, rows, inputs, dtype=dtype).requires_grad_(), normal(g, len(counts), outputs, inputs, dtype=dtype).requires_grad_()
    bias = normal(g, len(counts), outputs, dtype=dtype).requires_grad_()
    grad = normal(g, rows, outputs, dtype=dtype)
    y = tokens.grouped_linear(x, weight, offsets_of(counts), bias)
    gradients = torch.autograd.grad(y, (x, weight, bias), grad)
    exact = grouped_reference(x.detach(), weight.detach(), counts, bias.detach(), grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight", "bias")):
        near(value, expected, error, what)
    assert torch.equal(y, tokens.grouped_linear(x, weight, offsets_of(counts), bias))


@gpu
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (3, 5), (16, 32), (64, 64), (64, 56), (77, 130), (200, 33), (256, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_and_its_gradients(counts, inputs, outputs, dtype):
    say("grouped linear", counts, inputs, outputs, dtype)
    counts = COUNTS[counts]
    g = generator(inputs + len(counts))
    ungrouped = outputs % 7
    rows = sum(counts) + ungrouped
    x, weight = normal(g, rows, inputs, dtype=dtype).requires_grad_(), normal(g, len(counts), outputs, inputs, dtype=dtype).requires_grad_()
    bias = normal(g, len(counts), outputs, dtype=dtype).requires_grad_() if inputs % 2 else None
    grad = normal(g, rows, outputs, dtype=dtype)
    wanted = [t for t in (x, weight, bias) if t is not None]
    call = lambda: tokens.grouped_linear(x, weight, offsets_of(counts), bias)  # noqa: E731
    y = call()
    gradients = torch.autograd.grad(y, wanted, grad)
    exact = grouped_reference(x.detach(), weight.detach(), counts, bias.detach() if bias is not None else None, grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight", "bias")):
        near(value, expected, error, what)
    for a, b in zip(gradients, torch.autograd.grad(call(), wanted, grad)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("experts", [63, 64, 65, 128, 511, 512, 513, 4095, 4096, 4097, 5000])
def test_numbers_of_experts(experts):
    """A workgroup looks for its expert 64 at a time: numbers around the powers of 64, experts without rows among them."""
    say("numbers of experts", experts)
    g = generator(experts)
    counts = [(11 * e + experts) % 5 * (e % 3 != 1) + 70 * (e in (0, 63, 64, experts - 1)) for e in range(experts)]
    rows = sum(counts) + 3
    x, weight = normal(g, rows, 16, dtype=torch.float16).requires_grad_(), normal(g, experts, 8, 16, dtype=torch.float16).requires_grad_()
    grad = normal(g, rows, 8, dtype=torch.float16)
    y = tokens.grouped_linear(x, weight, offsets_of(counts))
    gradients = torch.autograd.grad(y, (x, weight), grad)
    exact = grouped_reference(x.detach(), weight.detach(), counts, None, grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight")):
        near(value, expected, error, what)


@gpu
@pytest.mark.parametrize("inputs,outputs", [(520, 264), (521, 263), (96, 136)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_many_experts(inputs, outputs, dtype):
    """Enough work for the largest tiles, with and without alignment; experts whose rows end anywhere in one."""
    say("many rows of many experts", inputs, outputs, dtype)
    g = generator(outputs)
    counts = [450 + (37 * e) % 140 for e in range(260)]
    counts[7], counts[100], counts[259] = 0, 1, 3000
    rows = sum(counts) + 5
    x, weight = normal(g, rows, inputs, dtype=dtype).requires_grad_(), normal(g, 260, outputs, inputs, dtype=dtype).requires_grad_()
    bias = normal(g, 260, outputs, dtype=dtype).requires_grad_()
    grad = normal(g, rows, outputs, dtype=dtype)
    y = tokens.grouped_linear(x, weight, offsets_of(counts), bias)
    gradients = torch.autograd.grad(y, (x, weight, bias), grad)
    exact = grouped_reference(x.detach(), weight.detach(), counts, bias.detach(), grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight", "bias")):
        near(value, expected, error, what)


@gpu
@pytest.mark.parametrize("stride", [(1 << 21) - 8, 1 << 21, (1 << 21) + 8, (1 << 22) + 1])
def test_grouped_linear_of_rows_far_apart(stride):
    """256 rows of a tile are reached with 32-bit offsets where they lie less than 2^21 entries apart; others are copied first."""
    say("rows far apart", stride)
    g = generator(stride)
    counts = [5, 0, 11]
    memory = torch.zeros(17 * stride + 64, dtype=torch.bfloat16, device="cuda")
    x = memory.as_strided((17, 48), (stride, 1))
    x.copy_(normal(g, 17, 48, dtype=torch.bfloat16))
    x.requires_grad_()
    weight, grad = normal(g, 3, 24, 48, dtype=torch.bfloat16).requires_grad_(), normal(g, 17, 24, dtype=torch.bfloat16)
    y = tokens.grouped_linear(x, weight, offsets_of(counts))
    gradients = torch.autograd.grad(y, (x, weight), grad)
    exact = grouped_reference(x.detach(), weight.detach(), counts, None, grad)
    for value, (expected, error), what in zip((y.detach(), *gradients), exact, ("y", "x", "weight")):
        near(value, expected, error, what)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_linear_of_other_strides(dtype):
    """Rows and matrices that lie apart, begin at odd addresses, or are one and the same; gradients of a shared matrix."""
    g = generator(11)
    counts = [70, 0, 200, 31]
    wide, stack = normal(g, 310, 200, dtype=dtype), normal(g, 4, 90, 101, dtype=dtype)
    for x in (wide[:, 1:65], wide[:, 3:68][::1], wide[5:, :64], wide.t()[:200].t()[:, :64]):
        x = x.detach()[:301].requires_grad_()
        n = x.shape[1]
        for weight in (stack[:, :, 1:1 + n], stack[:, 5:72, :n], stack[:1, :, :n].expand(4, 90, n), stack.transpose(1, 2)[:, :80, :n] if n <= 90 else stack[:, :, :n]):
            weight = weight.detach().requires_grad_()
            rows = x.shape[0]
            y = tokens.grouped_linear(x, weight, offsets_of(counts))
            grad = normal(g, rows, 2 * weight.shape[1], dtype=dtype)[:, 1:1 + weight.shape[1]]
            dx, dw = torch.autograd.grad(y, (x, weight), grad)
            exact = grouped_reference(x.detach(), weight.detach(), counts, None, grad)
            for value, (expected, error), what in zip((y.detach(), dx, dw), exact, ("y", "x", "weight")):
                near(value, expected, error, what)
    shared = normal(g, 90, 64, dtype=dtype).requires_grad_()
    x = normal(g, 301, 64, dtype=dtype)
    grad = normal(g, 301, 90, dtype=dtype)
    dw, = torch.autograd.grad(tokens.grouped_linear(x, shared.expand(4, 90, 64), offsets_of(counts)), shared, grad)
    _, _, (parts, error), _ = grouped_reference(x, shared.detach().expand(4, 90, 64), counts, None, grad)
    # (the experts' gradients are rounded, then torch adds them up in their type)
    near(dw, parts.sum(0), error.sum(0) + 8 * ROUNDING[dtype] * parts.abs().sum(0), "shared matrix")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_rows_of_one_expert_stay_with_it(dtype):
    """The tiles of other experts begin right behind: nothing of an infinite row or a NaN in it reaches them."""
    g = generator(12)
    counts = [37, 70, 5]
    x, weight, grad = normal(g, 120, 48, dtype=dtype), normal(g, 3, 40, 48, dtype=dtype), normal(g, 120, 40, dtype=dtype)
    clean = (x.clone(), grad.clone())
    x[37 + 69], grad[37 + 69] = float("inf"), float("nan")
    x[37], grad[37] = float("nan"), float("inf")
    x[112:], grad[112:] = float("nan"), float("nan")   # rows of no expert
    x.requires_grad_()
    weight.requires_grad_()
    bias = torch.zeros(3, 40, dtype=dtype, device="cuda").requires_grad_()
    y = tokens.grouped_linear(x, weight, offsets_of(counts), bias)
    dx, dw, db = torch.autograd.grad(y, (x, weight, bias), grad)
    exact = grouped_reference(clean[0], weight.detach(), counts, bias.detach(), clean[1])
    rows = [r for r in range(120) if r not in (37, 37 + 69)]
    near(y.detach()[rows], exact[0][0][rows], exact[0][1][rows], "y")
    near(dx[rows], exact[1][0][rows], exact[1][1][rows], "x")
    for value, (expected, error), what in ((dw, exact[2], "weight"), (db, exact[3], "bias")):
        near(value[[0, 2]], expected[[0, 2]], error[[0, 2]], what)
    assert bool(y[37].isnan().all()) and bool(db[1].isnan().all())
    # one infinite entry alone reaches its own output's gradients, no others
    grad = clean[1].clone()
    grad[40, 7] = float("inf")
    dw, db = torch.autograd.grad(tokens.grouped_linear(clean[0], weight, offsets_of(counts), bias), (weight, bias), grad)
    others = [i for i in range(40) if i != 7]
    near(dw[1][others], exact[2][0][1][others], exact[2][1][1][others], "other outputs")
    near(db[1][others], exact[3][0][1][others], exact[3][1][1][others], "other biases")
    assert not bool(db[1, 7].isfinite())


@gpu
def test_offsets_beyond_the_rows_are_limited_to_them():
    """Offsets that make no sense give no sensible rows, but every access stays within the tensors."""
    g = generator(13)
    x, weight = normal(g, 100, 16).requires_grad_(), normal(g, 4, 16, 16).requires_grad_()
    for offsets in ([0, 50, 1 << 30, 1 << 30, 1 << 30], [0, -5, -7, 1000, 20], [90, 80, 70, 60, 50]):
        y = tokens.grouped_linear(x, weight, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        torch.autograd.grad(y, (x, weight), torch.ones_like(y))
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ differences
@gpu
def test_gradients_are_slopes():
    """Central differences of a loss in every argument. Layers that are linear have no error but that of the arithmetic; of the layer norm's
    third derivative a step of 2^-6 leaves less than 1 %."""
    g = generator(20)
    index = torch.randint(-1, 6, (40,), device="cuda", generator=g)
    table, c = normal(g, 6, 12).requires_grad_(), normal(g, 40, 12)
    x, w, b, cn = normal(g, 10, 24).requires_grad_(), normal(g, 24).requires_grad_(), normal(g, 24).requires_grad_(), normal(g, 10, 24)
    xe, we, be, ce = normal(g, 30, 7).requires_grad_(), normal(g, 3, 5, 7).requires_grad_(), normal(g, 3, 5).requires_grad_(), normal(g, 30, 5)
    off = offsets_of([11, 0, 17])
    losses = [((table,), lambda: (tokens.embedding(index, table, 0.7) * c).double().sum()),
              ((x, w, b), lambda: (tokens.layer_norm(x, w, b) * cn).double().sum()),
              ((xe, we, be), lambda: (tokens.grouped_linear(xe, we, off, be) * ce).double().sum())]
    step = 2.0 ** -6
    for arguments, loss in losses:
        for argument, gradient in zip(arguments, torch.autograd.grad(loss(), arguments)):
            direction = normal(g, *argument.shape)
            with torch.no_grad():
                kept = argument.clone()
                argument.copy_(kept + step * direction)
                up = float(loss())
                argument.copy_(kept - step * direction)
                down = float(loss())
                argument.copy_(kept)
            slope = float((gradient.double() * direction.double()).sum())
            scale = float((gradient.double() * direction.double()).abs().sum())
            assert abs((up - down) / (2 * step) - slope) <= 0.01 * scale


# ------------------------------------------------------------------------------------------------ streams, graphs, autograd
def step_of_everything(table, index, w, b, weight, offsets, grad):
    y = tokens.grouped_linear(tokens.layer_norm(tokens.embedding(index, table, 2.0), w, b), weight, offsets)
    return (y, *torch.autograd.grad(y, (table, w, b, weight), grad))


def arguments_of_everything(seed=30):
    g = generator(seed)
    return [normal(g, 100, 64).requires_grad_(), torch.randint(0, 100, (9000,), device="cuda", generator=g), normal(g, 64).requires_grad_(),
            normal(g, 64).requires_grad_(), normal(g, 4, 48, 64).requires_grad_(), offsets_of([2000, 0, 4000, 3000]), normal(g, 9000, 48)]


@gpu
def test_calls_run_on_the_current_stream():
    arguments = arguments_of_everything()
    expected = [t.detach().clone() for t in step_of_everything(*arguments)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = [a.detach().clone().requires_grad_(a.requires_grad) for a in arguments]   # made on this stream: no other may read them yet
        results = step_of_everything(*late)
    stream.synchronize()
    for a, b in zip(results, expected):
        assert torch.equal(a, b)


@gpu
def test_steps_can_be_captured_and_replayed():
    arguments = arguments_of_everything()
    step_of_everything(*arguments)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step_of_everything(*arguments)
        order, offsets = tokens.group(arguments[1], 100)
    for turn in range(4):
        fresh = arguments_of_everything(40 + turn)
        with torch.no_grad():
            for a, f in zip(arguments, fresh):
                a.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*results, order, offsets), (*step_of_everything(*fresh), *tokens.group(fresh[1], 100))):
            assert torch.equal(a, b), turn


@gpu
def test_gradients_only_where_they_are_asked_for():
    table, index, w, b, weight, offsets, grad = arguments_of_everything()
    x = tokens.embedding(index, table.detach())
    assert not x.requires_grad
    only_w = tokens.layer_norm(x, w, b.detach())
    g_all = torch.autograd.grad(tokens.layer_norm(x.requires_grad_(), w, b), (x, w, b), torch.ones_like(x))
    assert torch.equal(torch.autograd.grad(only_w, w, torch.ones_like(only_w))[0], g_all[1])
    y = tokens.grouped_linear(x, weight, offsets)
    dx, dw = torch.autograd.grad(y, (x, weight), grad, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, grad, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(y, weight, grad)[0], dw)
    with torch.no_grad():
        assert not tokens.grouped_linear(x, weight, offsets).requires_grad


@gpu
def test_gradients_of_gradients_are_refused():
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(tokens.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated"):
        dx.sum().backward()


# ------------------------------------------------------------------------------------------------ refusals
@gpu
def test_arguments_that_do_not_fit_are_refused():
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
    for call, match in [
            (lambda: tokens.embedding(f(3), f(4, 5)), "index must hold"),
            (lambda: tokens.embedding(i32(3), f(4)), "2 dimensions"),
            (lambda: tokens.embedding(i32(3), f(4, 5, dtype=torch.float64)), "float, half or bfloat16"),
            (lambda: tokens.embedding(i32(3).cpu(), f(4, 5)), "GPU"),
            (lambda: tokens.group(f(3), 4), "index must hold"),
            (lambda: tokens.group(i32(3), -1), "number of groups"),
            (lambda: tokens.layer_norm(f(3, 4), f(5)), "must have 4 entries"),
            (lambda: tokens.layer_norm(f(3, 4), None, f(4, dtype=torch.float16)), "input's type or FLOAT"),
            (lambda: tokens.layer_norm(f(3, 4, dtype=torch.float16), f(4), f(4, dtype=torch.float16)), "one type"),
            (lambda: tokens.layer_norm(f(3, 4, dtype=torch.float64)), "float, half or bfloat16"),
            (lambda: tokens.grouped_linear(f(3, 4), f(2, 5, 6), i32(3)), "must have 4 entries"),
            (lambda: tokens.grouped_linear(f(3, 4), f(2, 5, 4), i32(2)), "must have 3 entries"),
            (lambda: tokens.grouped_linear(f(3, 4), f(2, 5, 4), i32(3).long()), "INT32"),
            (lambda: tokens.grouped_linear(f(3, 4), f(2, 5, 4, dtype=torch.float16), i32(3)), "must be of type FLOAT"),
            (lambda: tokens.grouped_linear(f(3, 4), f(2, 5, 4), i32(3), f(2, 4)), "must have 5 entries"),
            (lambda: tokens.grouped_linear(f(3, 0), f(2, 5, 0), i32(3)), "inputs and outputs"),
            (lambda: tokens.grouped_linear(f(3, 4), f(5, 4), i32(3)), "3 dimensions")]:
        with pytest.raises((qmlp.QmlpError, RuntimeError, ValueError, TypeError), match=match):
            call()


def test_tensors_on_the_host_are_refused():
    for call in (lambda: tokens.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 5)), lambda: tokens.layer_norm(torch.zeros(3, 4)),
                 lambda: tokens.group(torch.zeros(3, dtype=torch.int64), 2),
                 lambda: tokens.grouped_linear(torch.zeros(3, 4), torch.zeros(2, 5, 4), torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


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


def test_c_interface_refuses_before_any_launch():
    """Descriptors that do not fit end in a status and a message; nothing of them is read (these calls need no device)."""
    lib, F, H, B, I = _lib.lib, _lib.QMLP_FLOAT, _lib.QMLP_HALF, _lib.QMLP_BFLOAT16, _lib.QMLP_INT32
    x, y = descriptor(F, 4, 6), descriptor(F, 4, 6)
    none = _lib.TensorDesc()
    norm = lambda *a: lib.qmlp_tokens_layer_norm(*a, 1e-5, y, none, none, None)  # noqa: E731
    refused(norm(descriptor(F, 4, 6, strides=(12, 2)), none, none), "consecutive")
    refused(norm(descriptor(F, 4, 6, strides=(-6, 1)), none, none), "negative stride")
    refused(norm(descriptor(_lib.QMLP_DOUBLE, 4, 6), none, none), "float, half or bfloat16")
    refused(norm(descriptor(17, 4, 6), none, none), "unknown tensor precision")
    refused(norm(x, descriptor(F, 7), none), "must have 6 entries")
    refused(norm(none, none, none), "undefined")
    refused(lib.qmlp_tokens_layer_norm(x, none, none, 1e-5, descriptor(F, 4, 6, strides=(3, 1)), none, none, None), "share memory")
    refused(lib.qmlp_tokens_layer_norm_adjoint(x, none, none, none, y, y, none, none, None, None), "mean is undefined")
    mean = descriptor(F, 4)
    refused(lib.qmlp_tokens_layer_norm_adjoint(x, none, mean, mean, y, none, descriptor(F, 6), none, None, None), "bytes of memory")
    refused(lib.qmlp_tokens_layer_norm_adjoint(x, none, mean, mean, y, none, descriptor(F, 6), none, 264, None), "aligned")
    refused(lib.qmlp_tokens_embedding(descriptor(F, 4), descriptor(F, 9, 6), 1.0, y, None), "index must hold")
    refused(lib.qmlp_tokens_embedding(descriptor(I, 5), descriptor(F, 9, 6), 1.0, y, None), "must have 5 entries")
    refused(lib.qmlp_tokens_embedding(descriptor(I, 4), descriptor(B, 9, 6), 1.0, y, None), "must be of type BFLOAT16")
    refused(lib.qmlp_tokens_embedding_adjoint(descriptor(I, 4), y, 1.0, descriptor(F, 9, 6), None, None), "bytes of memory")
    refused(lib.qmlp_tokens_group(descriptor(I, 4), -1, descriptor(I, 4), descriptor(I, 4), None, None), "must not be negative")
    refused(lib.qmlp_tokens_group(descriptor(I, 4), 3, descriptor(I, 4), descriptor(I, 3), None, None), "must have 4 entries")
    w, off = descriptor(F, 3, 5, 6), descriptor(I, 4)
    refused(lib.qmlp_tokens_grouped_linear(x, w, off, none, y, None, None), "must have 5 entries")
    refused(lib.qmlp_tokens_grouped_linear(x, descriptor(H, 3, 5, 6), off, none, y, None, None), "must be of type FLOAT")
    refused(lib.qmlp_tokens_grouped_linear(x, w, descriptor(F, 4), none, y, None, None), "must be of type INT32")
    dy = descriptor(F, 4, 5)
    refused(lib.qmlp_tokens_grouped_linear_adjoint(x, w, off, dy, none, descriptor(F, 3, 5, 6, strides=(60, 12, 1)), none, None, None), "contiguous")
    for call in (lambda b: lib.qmlp_tokens_group_memory(-1, 4, b), lambda b: lib.qmlp_tokens_group_memory(1 << 31, 4, b),
                 lambda b: lib.qmlp_tokens_embedding_adjoint_memory(4, -1, 4, b), lambda b: lib.qmlp_tokens_layer_norm_adjoint_memory(-1, 4, b),
                 lambda b: lib.qmlp_tokens_grouped_linear_adjoint_memory(-1, 1, 1, 1, b)):
        refused(call(ctypes.byref(ctypes.c_size_t())), "must not be negative")
    refused(lib.qmlp_tokens_precompile(_lib.QMLP_DOUBLE), "precision must be")


def test_other_entry_points_refuse_the_further_types():
    """Networks and encodings know float, half and double alone."""
    out = ctypes.c_void_p()
    assert _lib.lib.qmlp_activation_create(b"relu", ctypes.byref(out)) == 0
    for p in (_lib.QMLP_BFLOAT16, _lib.QMLP_INT32, _lib.QMLP_INT64):
        d = descriptor(p, 4, 6)
        refused(_lib.lib.qmlp_activation_forward(out, d, d, None), "unknown tensor precision")
    _lib.check(_lib.lib.qmlp_activation_destroy(out))
    with pytest.raises(TypeError):
        _lib.desc(torch.zeros(3, dtype=torch.bfloat16))


def test_memory_sizes_grow_with_the_work():
    size = ctypes.c_size_t()
    def of(function, *arguments):
        _lib.check(function(*arguments, ctypes.byref(size)))
        return size.value
    lib = _lib.lib
    assert of(lib.qmlp_tokens_group_memory, 8192, 100) == 0   # one workgroup's registers
    assert of(lib.qmlp_tokens_group_memory, 0, 0) == 0
    assert 0 < of(lib.qmlp_tokens_group_memory, 1 << 20, 8) < of(lib.qmlp_tokens_group_memory, 1 << 20, 4096)
    assert of(lib.qmlp_tokens_embedding_adjoint_memory, 1000, 50, 64) < of(lib.qmlp_tokens_embedding_adjoint_memory, 100000, 50, 64)
    assert of(lib.qmlp_tokens_layer_norm_adjoint_memory, 0, 64) == 0
    assert of(lib.qmlp_tokens_layer_norm_adjoint_memory, 1, 64) >= 2 * 64 * 4
    assert of(lib.qmlp_tokens_grouped_linear_adjoint_memory, 0, 4, 64, 64) == 0
    assert of(lib.qmlp_tokens_grouped_linear_memory, 4096, 4, 64, 64) == 0 and of(lib.qmlp_tokens_grouped_linear_memory, 4, 4, 4096, 64) > 0
