"""The router and the rows of tokens to their experts and back (qmlp.tokens) against their definitions in 64 bits.

Tolerances: sums of n terms in 32 bits are off by at most n 2^-23 of the sum of their magnitudes, a result is rounded once to its type.
"""
import ctypes
import importlib.util
import os

import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

import qmlp
from qmlp import _lib, tokens
from token_helpers import DTYPES, U, Margins, described, descriptor, generator, near, normal, refused, say, skip_warming

gpu = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def no_warming(request):
    skip_warming(request)


# ------------------------------------------------------------------------------------------------ places of groups
@gpu
@pytest.mark.parametrize("groups", [0, 1, 8, 300, 4399, 4400, 70000])
@pytest.mark.parametrize("rows", [0, 1, 65, 8192, 8193, 70001])
def test_places_are_the_inverse_of_the_order(rows, groups):
    say("places", rows, groups)
    rng = np.random.default_rng(rows + groups)
    index = torch.from_numpy(rng.integers(-2, groups + 3, rows)).cuda()
    order, offsets, places = tokens.group(index, groups, places=True)
    plain_order, plain_offsets = tokens.group(index, groups)
    assert torch.equal(order, plain_order) and torch.equal(offsets, plain_offsets)
    expected = torch.empty(rows, dtype=torch.int32, device="cuda")
    expected[order.long()] = torch.arange(rows, dtype=torch.int32, device="cuda")
    expected = torch.where((index >= 0) & (index < groups), expected, -1 - expected)
    assert torch.equal(places, expected)


@gpu
def test_places_have_the_shape_of_the_index():
    index = torch.randint(-1, 5, (6, 7, 2), device="cuda").transpose(0, 1)
    order, _, places = tokens.group(index, 5, places=True)
    assert places.shape == (7, 6, 2)
    flat = torch.where(places >= 0, places, -1 - places).flatten()
    assert torch.equal(order[flat.long()], torch.arange(84, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------------------ router
def route_reference(logits, chosen, normalised, grad):
    """Weights, their error, index, gradient of the logits, its error."""
    l = logits.double()
    experts = l.shape[1]
    top = l.max(1, keepdim=True)[0]
    any_ = top > -INF
    away = torch.where(any_, l - torch.where(any_, top, 0.0), -INF)
    e = torch.where(any_, torch.exp(away), 0.0)
    values, index = torch.sort(l, dim=1, descending=True, stable=True)
    values, index = values[:, :chosen], index[:, :chosen]
    taken = values > -INF
    held = torch.zeros_like(l).scatter_(1, index, taken.double())
    total = torch.where(any_, ((e * held) if normalised else e).sum(1, keepdim=True), 1.0)
    p = (e * held if normalised else e) / total
    # the difference to the largest logit is rounded, exp to 2 units, the sum has as many terms as there are experts
    spread = torch.where(away > -200, -away, 0.0)   # (exp(-200) is below the smallest number)
    relative = (spread + spread.max(1, keepdim=True)[0] + experts + chosen + 16) * U
    w = torch.where(taken, torch.gather(p, 1, index), 0.0)
    e_w = w * torch.gather(relative, 1, index) + 2.0 ** -126
    g = torch.where(taken, grad.double(), 0.0)
    full = torch.zeros_like(l).scatter_(1, index, g)
    inner, size = (p * full).sum(1, keepdim=True), (p * full).abs().sum(1, keepdim=True)
    dl = p * (full - inner)
    e_dl = p * 2 * relative.max(1, keepdim=True)[0] * (full.abs() + size + inner.abs()) + 2.0 ** -126
    if normalised:
        dl = dl * held
    return w, e_w, torch.where(taken, index, -1).int(), dl, e_dl


@gpu
@pytest.mark.parametrize("experts", [1, 2, 7, 8, 31, 32, 33, 64, 65, 128, 129, 256, 257, 500, 512, 513, 1000, 1024, 1025, 5000])
@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("dtype", DTYPES)
def test_route_and_its_gradient(rows, experts, dtype):
    say("route", rows, experts, dtype)
    g = generator(experts + rows)
    logits = 2 * normal(g, rows, experts)
    if rows > 1:   # many equal logits in some rows
        logits[1::3] = torch.round(logits[1::3])
    logits = logits.to(dtype).requires_grad_()
    for chosen in sorted({1, min(2, experts), min(5, experts), min(8, experts), min(17, experts), min(64, experts)}):
        for normalised in (False, True):
            grad = normal(g, rows, chosen, dtype=dtype)
            weights, index = tokens.route(logits, chosen, normalised)
            dlogits, = torch.autograd.grad(weights, logits, grad)
            w, e_w, expected, dl, e_dl = route_reference(logits.detach(), chosen, normalised, grad)
            assert index.dtype == torch.int32 and not index.requires_grad and torch.equal(index, expected)
            near(weights.detach(), w, e_w, "weights")
            near(dlogits, dl, e_dl, "gradient")
            again = tokens.route(logits, chosen, normalised)
            assert torch.equal(again[0], weights) and torch.equal(torch.autograd.grad(again[0], logits, grad)[0], dlogits)


@gpu
@pytest.mark.parametrize("experts", [4, 30, 100, 700, 1500])
@pytest.mark.parametrize("normalised", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_experts_are_taken_by_no_row(experts, normalised, dtype):
    """Fewer experts than are chosen, none at all, and masks of the lowest finite number, which are logits as others."""
    say("masked", experts, normalised, dtype)
    g = generator(experts)
    logits = normal(g, 60, experts)
    logits[torch.rand(60, experts, device="cuda", generator=g) < 0.5] = -INF
    logits = logits.to(dtype)
    logits[3] = -INF
    logits[4] = -INF
    logits[4, experts - 1] = 0.5
    logits[5] = torch.finfo(dtype).min
    logits[6, 1:] = torch.finfo(dtype).min
    logits[7], logits[7, 0] = torch.finfo(dtype).min, -INF
    logits[8] = torch.finfo(dtype).max
    logits[9, 0::2], logits[9, 1::2] = 0.0, -0.0   # equal: the first ones
    logits.requires_grad_()
    grad = normal(g, 60, 4, dtype=dtype)
    weights, index = tokens.route(logits, 4, normalised)
    dlogits, = torch.autograd.grad(weights, logits, grad)
    w, e_w, expected, dl, e_dl = route_reference(logits.detach(), 4, normalised, grad)
    assert torch.equal(index, expected)
    assert index[3].tolist() == [-1] * 4 and index[4].tolist() == [experts - 1, -1, -1, -1] and index[9].tolist() == [0, 1, 2, 3]
    assert weights[3].tolist() == [0.0] * 4 and float(weights[4, 0].detach()) == 1
    near(weights.detach(), w, e_w, "weights")
    near(dlogits, dl, e_dl, "gradient")
    assert not bool(dlogits[3].any())


@gpu
@pytest.mark.parametrize("experts", [8, 33, 200, 500, 1024, 1025])
@pytest.mark.parametrize("normalised", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_below_the_normal_numbers(experts, normalised, dtype):
    """Shares from 2^-115 down to the smallest number there is: the exponential and its quotient are each off by half of 2^-149 besides what they are
    relative to their size. In gradients up to 1024 experts count shares below 2^-126 as 0."""
    logits = torch.full((3, experts), -200.0)
    logits[0, :8] = torch.tensor([0.0, -80.0, -87.25, -87.5, -90.0, -95.0, -100.0, -103.0])
    logits[1, :8] = torch.tensor([-0.5, -60.0, -86.0, -88.0, -93.0, -97.0, -101.5, -102.5])
    logits[2, -8:] = torch.tensor([-102.0, -99.0, -98.0, -94.0, -92.0, -89.0, -87.0, 1.0])
    logits = logits.to(dtype).cuda().requires_grad_()
    grad = (torch.tensor([1.0, -2.0, 3.0, -1.0, 2.0, -3.0, 1.0, 4.0]) * torch.tensor([1.0] + [2.0 ** 30] * 7)).to(dtype).expand(3, 8).contiguous().cuda()
    weights, index = tokens.route(logits, 8, normalised)
    dlogits, = torch.autograd.grad(weights, logits, grad)
    w, e_w, expected, dl, _ = route_reference(logits.detach(), 8, normalised, grad)
    assert torch.equal(index, expected)
    near(weights.detach(), w, e_w - 2.0 ** -126 + 2.0 ** -150, "weights")
    relative = 2 * (220 + experts + 8 + 16) * U
    l = logits.detach().double()
    p = torch.exp(l - l.max(1, keepdim=True)[0])
    p = p / torch.gather(p, 1, index.long()).sum(1, keepdim=True) if normalised else p / p.sum(1, keepdim=True)
    full = torch.zeros_like(l).scatter_(1, index.long(), grad.double())
    size = full.abs() + 2 * (p * full).abs().sum(1, keepdim=True)
    near(dlogits, dl, (p * relative + (2.0 ** -126 if experts <= 1024 else 2.0 ** -149)) * size, "gradient")
    if dtype == torch.float32:
        assert int((weights > 0).sum()) == 24 and int((weights < 2.0 ** -126).sum()) == 17


@gpu
@pytest.mark.parametrize("experts", [5, 64, 300, 1024, 3000])
def test_rows_that_are_not_numbers_stay_alone(experts):
    g = generator(experts + 1)
    logits = normal(g, 50, experts)
    clean = logits.clone()
    logits[11, 2], logits[20, experts - 1], logits[30, 0] = float("nan"), INF, -float("nan")
    logits.requires_grad_()
    clean.requires_grad_()
    grad = normal(g, 50, 3)
    for normalised in (False, True):
        weights, index = tokens.route(logits, 3, normalised)
        dlogits, = torch.autograd.grad(weights, logits, grad)
        expected, order = tokens.route(clean, 3, normalised)
        dclean, = torch.autograd.grad(expected, clean, grad)
        for r in (11, 20, 30):
            assert bool(weights[r].isnan().any()) and bool(dlogits[r].isnan().any())
            assert len(set(index[r].tolist())) == 3 and 0 <= int(index[r].min()) and int(index[r].max()) < experts
        assert int(index[11, 0]) == 2 and int(index[20, 0]) == experts - 1 and int(index[30, 0]) == 0
        keep = [r for r in range(50) if r not in (11, 20, 30)]
        assert torch.equal(weights[keep], expected[keep]) and torch.equal(index[keep], order[keep]) and torch.equal(dlogits[keep], dclean[keep])


@gpu
def test_route_takes_any_shape_and_stride():
    g = generator(3)
    wide = normal(g, 9, 40, 70)
    for logits in (wide[..., 5:38], wide[::2, :, 1:], wide.transpose(0, 2), wide[:1].expand(9, 40, 70), wide[0, 0], wide[:0]):
        logits = logits.detach().requires_grad_()
        weights, index = tokens.route(logits, 3)
        assert weights.shape == index.shape == (*logits.shape[:-1], 3)
        grad = normal(g, *weights.shape, 2)[..., 0]
        dlogits, = torch.autograd.grad(weights, logits, grad)
        assert dlogits.shape == logits.shape
        w, e_w, expected, dl, e_dl = route_reference(logits.detach().reshape(-1, logits.shape[-1]), 3, False, grad.reshape(-1, 3)) if logits.numel() else [None] * 5
        if w is not None:
            assert torch.equal(index.reshape(-1, 3), expected)
            near(weights.detach().reshape(-1, 3), w, e_w, "weights")
            near(dlogits.reshape(-1, logits.shape[-1]), dl, e_dl, "gradient")


@gpu
@pytest.mark.parametrize("rows,experts,chosen", [(65536 * 32 + 33, 3, 2), (4096 + 5, 1025, 3)])
@pytest.mark.parametrize("normalised", [False, True])
def test_more_rows_than_workgroups_of_a_launch(rows, experts, chosen, normalised):
    """The kernels go on in steps of the grid: 65536 workgroups of 32 rows, 4096 of a row where no wavefront holds one."""
    g = generator(rows)
    logits = normal(g, rows, experts, dtype=torch.float16).requires_grad_()
    grad = normal(g, rows, chosen, dtype=torch.float16)
    weights, index = tokens.route(logits, chosen, normalised)
    dlogits, = torch.autograd.grad(weights, logits, grad)
    w, e_w, expected, dl, e_dl = route_reference(logits.detach(), chosen, normalised, grad)
    assert torch.equal(index, expected)
    near(weights.detach(), w, e_w, "weights")
    near(dlogits, dl, e_dl, "gradient")


# ------------------------------------------------------------------------------------------------ rows to experts and back
def places_of(g, tokens_, chosen, dropped=0.1):
    index = torch.randint(0, 6, (tokens_, chosen), device="cuda", generator=g)
    index[torch.rand(tokens_, chosen, device="cuda", generator=g) < dropped] = -1
    if tokens_ > 2:
        index[2] = -1   # a token without experts
    return tokens.group(index, 6, places=True)[2]


def rows_reference(places, C):
    """Row and token of every place that belongs to an expert, and the rows of the others."""
    flat = places.long().flatten()
    token = torch.arange(places.shape[0], device="cuda").repeat_interleave(places.shape[1])
    has = flat >= 0
    return flat[has], token[has], has, -1 - flat[~has]


@gpu
@pytest.mark.parametrize("channels", [1, 3, 8, 31, 64, 100, 512, 777, 2048, 5000])
@pytest.mark.parametrize("tokens_,chosen", [(0, 2), (1, 1), (3, 2), (65, 8), (700, 3), (40, 17)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_to_experts_and_back(tokens_, chosen, channels, dtype):
    say("rows", tokens_, chosen, channels, dtype)
    g = generator(tokens_ + channels)
    places = places_of(g, tokens_, chosen)
    place, token, has, without = rows_reference(places, channels)
    x = normal(g, tokens_, channels, dtype=dtype).requires_grad_()
    drows = normal(g, tokens_ * chosen, channels, dtype=dtype)
    drows[without] = float("nan")   # (no part of any gradient)
    rows = tokens.dispatch(x, places)
    dx, = torch.autograd.grad(rows, x, drows)
    expected = torch.zeros_like(drows)
    expected[place] = x.detach()[token]
    assert torch.equal(rows, expected)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")  # noqa: E731
    exact, size = zeros(tokens_, channels).index_add_(0, token, drows[place].double()), zeros(tokens_, channels).index_add_(0, token, drows[place].double().abs())
    near(dx, exact, chosen * U * size, "gradient of the tokens")

    rows = normal(g, tokens_ * chosen, channels, dtype=dtype)
    rows[without] = float("nan")
    rows.requires_grad_()
    for weight_type in {torch.float32, dtype}:
        weights = normal(g, tokens_, chosen, dtype=weight_type).requires_grad_()
        residual = normal(g, tokens_, channels, dtype=dtype).requires_grad_()
        dy = normal(g, tokens_, channels, dtype=dtype)
        y = tokens.combine(rows, places, weights, residual)
        drows, dweights, dresidual = torch.autograd.grad(y, (rows, weights, residual), dy)
        w, r, d = weights.detach().double().flatten()[has][:, None], rows.detach().double()[place], dy.double()[token]
        exact = residual.detach().double().index_add_(0, token, w * r)
        size = residual.detach().double().abs().index_add_(0, token, (w * r).abs())
        near(y.detach(), exact, (chosen + 2) * U * size, "combined")
        exact = zeros(tokens_ * chosen, channels)
        exact[place] = w * d
        near(drows, exact, U * exact.abs(), "gradient of the rows")
        exact, size = zeros(tokens_ * chosen), zeros(tokens_ * chosen)
        exact[has], size[has] = (d * r).sum(1), (d * r).abs().sum(1)
        near(dweights.flatten(), exact, (channels + 4) * U * size, "gradient of the weights")
        assert torch.equal(dresidual, dy) and dweights.dtype == weight_type
        again = tokens.combine(rows, places, weights, residual)
        assert torch.equal(again, y)
        for a, b in zip(torch.autograd.grad(again, (rows, weights), dy), (drows, dweights)):
            assert torch.equal(a, b)
        # one gradient without the others
        assert torch.equal(torch.autograd.grad(tokens.combine(rows, places, weights.detach()), rows, dy)[0], drows)
        assert torch.equal(torch.autograd.grad(tokens.combine(rows.detach(), places, weights), weights, dy)[0], dweights)
    y = tokens.combine(rows, places)
    drows, = torch.autograd.grad(y, rows, dy)
    exact = zeros(tokens_, channels).index_add_(0, token, r)
    near(y.detach(), exact, chosen * U * zeros(tokens_, channels).index_add_(0, token, r.abs()), "sum")
    expected = torch.zeros_like(drows)
    expected[place] = dy[token]
    assert torch.equal(drows, expected)


@gpu
@pytest.mark.parametrize("channels", [40, 520, 1023, 1024, 1032])
@pytest.mark.parametrize("tokens_", [2048, 2049])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_tokens_that_are_shared_out_and_not(tokens_, channels, dtype):
    """Tokens and channels at which wavefronts begin to share the rows of a token, or to take them one after the other."""
    test_rows_to_experts_and_back(tokens_, 3, channels, dtype)


@gpu
def test_rows_of_other_shapes_and_strides():
    g = generator(5)
    wide = normal(g, 6, 7, 90)
    index = torch.randint(-1, 4, (7, 6, 3), device="cuda", generator=g).transpose(0, 1)
    _, _, places = tokens.group(index, 4, places=True)
    strided = torch.zeros(6, 7, 5, dtype=torch.int32, device="cuda")
    strided[..., 1:4] = places
    for p in (places, strided[..., 1:4], places.transpose(0, 1).contiguous().transpose(0, 1), places.flip(2).contiguous().flip(2)):
        for x in (wide[..., 3:60], wide.transpose(0, 1)[:, :, :50].transpose(0, 1), wide[..., ::2], wide[:1].expand(6, 7, 90)):
            x = x.detach().requires_grad_()
            C = x.shape[-1]
            rows = tokens.dispatch(x, p)
            place, token, has, _ = rows_reference(p.reshape(-1, 3), C)
            expected = torch.zeros(126, C, device="cuda")
            expected[place] = x.detach().reshape(-1, C)[token]
            assert torch.equal(rows, expected)
            dx, = torch.autograd.grad(rows, x, torch.ones(1, 1, device="cuda").expand(126, C))
            assert torch.equal(dx, (p >= 0).sum(-1, keepdim=True).float().expand(6, 7, C))
            weights = normal(g, 7, 6, 3).transpose(0, 1).detach().requires_grad_()
            wide_rows = normal(g, 126, 2 * C)[:, 1:C + 1].requires_grad_()
            y = tokens.combine(wide_rows, p, weights, x)
            assert y.shape == x.shape
            drows, dweights, dx = torch.autograd.grad(y, (wide_rows, weights, x), torch.ones(1, 1, 1, device="cuda").expand(6, 7, C))
            w = weights.detach().reshape(-1)[has]
            expected = torch.zeros(126, C, device="cuda")
            expected[place] = w[:, None].expand(-1, C)
            assert torch.equal(drows, expected) and dweights.shape == weights.shape and torch.equal(dx, torch.ones_like(dx))


@gpu
def test_rows_of_more_than_two_to_the_31_entries():
    """Rows whose first entries have no 32-bit offset."""
    tokens_, channels = (1 << 19) + 3, 2048
    places = torch.arange(2 * tokens_, dtype=torch.int32, device="cuda").flip(0).view(tokens_, 2).contiguous()
    x = torch.zeros(tokens_, channels, dtype=torch.float16, device="cuda")
    x[0], x[-1] = 3, 5
    x.requires_grad_()
    rows = tokens.dispatch(x, places)
    assert bool((rows[-2:] == 3).all()) and bool((rows[:2] == 5).all()) and int(torch.count_nonzero(rows)) == 4 * channels
    weights = torch.tensor([0.5, 2.0], device="cuda").expand(tokens_, 2)
    y = tokens.combine(rows.detach().requires_grad_(), places, weights)
    assert bool((y[0] == 7.5).all()) and bool((y[-1] == 12.5).all())
    dx, = torch.autograd.grad(rows, x, rows)
    assert bool((dx[0] == 6).all()) and bool((dx[-1] == 10).all()) and int(torch.count_nonzero(dx)) == 2 * channels
    drows, = torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[0][0].variable])
    assert bool((drows[-1] == 0.5).all()) and bool((drows[0] == 2).all())


@gpu
def test_more_tokens_than_workgroups_of_a_launch():
    """2^20 workgroups of 32 tokens, and a second turn."""
    tokens_ = (1 << 25) + 37
    places = torch.arange(tokens_, dtype=torch.int32, device="cuda").flip(0).view(tokens_, 1).contiguous()
    x = (torch.arange(tokens_, device="cuda") % 251).half().view(tokens_, 1).requires_grad_()
    rows = tokens.dispatch(x, places)
    assert torch.equal(rows.detach(), x.detach().flip(0))
    dx, = torch.autograd.grad(rows, x, x.detach())
    assert torch.equal(dx, x.detach().flip(0))
    r, w = rows.detach().requires_grad_(), (torch.arange(tokens_, device="cuda") % 4).half().view(tokens_, 1).requires_grad_()
    y = tokens.combine(r, places, w)
    assert torch.equal(y.detach(), w.detach() * x.detach())   # (products of numbers of 8 and 2 bits: exact)
    drows, dweights = torch.autograd.grad(y, (r, w), x.detach())
    assert torch.equal(drows, (w.detach() * x.detach()).flip(0))
    assert torch.equal(dweights, (x.detach().float() ** 2).half())   # (below 2^16; one rounding)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("channels", [3, 40, 777])
def test_places_that_make_no_sense_write_nothing_beside_the_results(dtype, channels):
    """Places of rows that are not there are left out, the same place twice is written twice: nothing beside rows and results is touched."""
    say("places", dtype, channels)
    lib, tokens_, chosen = _lib.lib, 50, 3
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    none = _lib.TensorDesc()
    x, rows_in = torch.ones(tokens_, channels, dtype=dtype, device="cuda"), torch.ones(tokens_ * chosen, channels, dtype=dtype, device="cuda")
    weights = torch.ones(tokens_, chosen, device="cuda")
    for value in (150, 2 ** 31 - 1, -2 ** 31, -151, 7, -8):
        margins = Margins(8)
        places = torch.full((tokens_, chosen), value, dtype=torch.int32, device="cuda")
        rows, drows = margins.tensor(dtype, tokens_ * chosen, channels), margins.tensor(dtype, tokens_ * chosen, channels)
        y, dw = margins.tensor(dtype, tokens_, channels), margins.tensor(torch.float32, tokens_, chosen)
        p = described(places)
        _lib.check(lib.qmlp_tokens_dispatch(described(x), p, described(rows), stream))
        _lib.check(lib.qmlp_tokens_combine(described(rows_in), p, described(weights), none, described(y), stream))
        _lib.check(lib.qmlp_tokens_combine_adjoint(described(rows_in), p, described(weights), described(x), described(drows), described(dw), stream))
        torch.cuda.synchronize()
        margins.untouched()
        expected = 3.0 if value == 7 else 0.0
        assert bool((y == expected).all()) and bool((dw == (channels if value == 7 else 0)).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,experts,chosen", [(1, 1, 1), (33, 7, 3), (70, 65, 64), (9, 1025, 2)])
def test_nothing_beside_the_results_of_the_router_is_written(dtype, rows, experts, chosen):
    lib = _lib.lib
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    margins = Margins(8)
    logits, grad = torch.randn(rows, experts, device="cuda").to(dtype), torch.randn(rows, chosen, device="cuda").to(dtype)
    weights, index, dlogits = margins.tensor(dtype, rows, chosen), margins.tensor(torch.int32, rows, chosen), margins.tensor(dtype, rows, experts)
    order, offsets, places = margins.tensor(torch.int32, rows * chosen), margins.tensor(torch.int32, experts + 1), margins.tensor(torch.int32, rows * chosen)
    _lib.check(lib.qmlp_tokens_route(described(logits), 0, described(weights), described(index), stream))
    _lib.check(lib.qmlp_tokens_route_adjoint(described(logits), described(index), described(grad), 0, described(dlogits), stream))
    size = ctypes.c_size_t()
    _lib.check(lib.qmlp_tokens_group_memory(rows * chosen, experts, ctypes.byref(size)))
    _lib.check(lib.qmlp_tokens_group_places(described(index.view(-1)), experts, described(order), described(offsets), described(places),
                                            margins.bytes(size.value), stream))
    torch.cuda.synchronize()
    margins.untouched()
    for wrong in (experts, -1, 2 ** 31 - 1, -2 ** 31):   # an index that names no expert has no part
        other = torch.full_like(index, wrong)
        _lib.check(lib.qmlp_tokens_route_adjoint(described(logits), described(other), described(grad), 0, described(dlogits), stream))
        torch.cuda.synchronize()
        margins.untouched()
        assert not bool(dlogits.any())


# ------------------------------------------------------------------------------------------------ together
def layer_of_experts(x, logits, first, second, chosen, normalised):
    """Router, sort, rows to the experts, their two layers, and back on top of the tokens."""
    weights, index = tokens.route(logits, chosen, normalised)
    _, offsets, places = tokens.group(index, first.shape[0], places=True)
    rows = torch.relu(tokens.grouped_linear(tokens.dispatch(x, places), first, offsets))
    return tokens.combine(tokens.grouped_linear(rows, second, offsets), places, weights, x)


def arguments_of_a_layer(seed, dtype=torch.float32):
    g = generator(seed)
    x, logits = normal(g, 300, 40, dtype=dtype), normal(g, 300, 6, dtype=dtype)
    logits[torch.rand(300, 6, device="cuda", generator=g) < 0.2] = -INF
    logits[17] = -INF
    first, second = (0.2 * normal(g, 6, 56, 40)).to(dtype), (0.2 * normal(g, 6, 40, 56)).to(dtype)
    return [t.requires_grad_() for t in (x, logits, first, second)] + [normal(g, 300, 40, dtype=dtype)]


def plain_layer(x, logits, first, second, chosen, normalised):
    """Every expert on every token, in 64 bits."""
    x, logits, first, second = (t.double() for t in (x, logits, first, second))
    index = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :chosen]
    held = torch.zeros_like(logits).scatter_(1, index, 1.0) * (logits > -INF)
    e = torch.exp(torch.where(logits > -INF, logits, -1e9)) * (logits > -INF)
    total = (e * held if normalised else e).sum(1, keepdim=True)
    w = e * held / torch.where(total > 0, total, 1.0)
    hidden = torch.relu(torch.stack([x @ f.T for f in first], 1))
    return x + (w[..., None] * torch.stack([hidden[:, e] @ second[e].T for e in range(len(second))], 1)).sum(1)


@gpu
@pytest.mark.parametrize("normalised", [False, True])
def test_a_layer_of_experts_is_that_of_plain_layers(normalised):
    x, logits, first, second, grad = arguments_of_a_layer(1)
    y = layer_of_experts(x, logits, first, second, 2, normalised)
    wanted = (x, logits, first, second)
    gradients = torch.autograd.grad(y, wanted, grad)
    expected = plain_layer(*wanted, 2, normalised)
    # sums of some hundred terms one behind the other, none of whose partial sums is above 2^10 of the results' size: 2^10 2^-23 is 2^-13
    torch.testing.assert_close(y.double(), expected, rtol=2.0 ** -13, atol=2.0 ** -13)
    for a, e in zip(gradients, torch.autograd.grad(expected, wanted, grad.double())):
        torch.testing.assert_close(a, e, rtol=2.0 ** -13, atol=2.0 ** -13 * float(e.abs().max()))
    assert torch.equal(y[17], x[17])   # a token without experts passes by


@gpu
@pytest.mark.parametrize("normalised", [False, True])
def test_gradients_are_slopes(normalised):
    """Central differences of a loss in every argument; a step of 2^-8 leaves less than 1 % of the softmax's third derivative."""
    g = generator(20)
    logits = normal(g, 20, 9)
    logits = (logits + 0.2 * torch.arange(9, device="cuda")).requires_grad_()   # (no two of a row change places)
    places = places_of(g, 20, 3)
    x, rows, weights, residual = (normal(g, *s).requires_grad_() for s in ((20, 12), (60, 12), (20, 3), (20, 12)))
    cw, cr, cy = normal(g, 20, 3), normal(g, 60, 12), normal(g, 20, 12)
    step = 2.0 ** -8
    gaps = torch.sort(logits.detach(), 1)[0].diff(dim=1)
    keep = (gaps.min(1)[0] > 12 * step)[:, None].float()   # rows whose order the step could change have no part
    losses = [((logits,), lambda: (tokens.route(logits, 3, normalised)[0] * cw * keep).double().sum()),
              ((x,), lambda: (tokens.dispatch(x, places) * cr).double().sum()),
              ((rows, weights, residual), lambda: (tokens.combine(rows, places, weights, residual) * cy).double().sum())]
    assert float(keep.sum()) >= 5
    for arguments, loss in losses:
        for argument, gradient in zip(arguments, torch.autograd.grad(loss(), arguments)):
            direction = normal(g, *argument.shape).clamp(-5, 5)
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


@gpu
def test_calls_run_on_the_current_stream():
    arguments = arguments_of_a_layer(30)
    run = lambda x, logits, first, second, grad: (  # noqa: E731
        lambda y: (y, *torch.autograd.grad(y, (x, logits, first, second), grad)))(layer_of_experts(x, logits, first, second, 2, True))
    expected = [t.detach().clone() for t in run(*arguments)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = [a.detach().clone().requires_grad_(a.requires_grad) for a in arguments]   # made on this stream: no other may read them yet
        results = run(*late)
    stream.synchronize()
    for a, b in zip(results, expected):
        assert torch.equal(a, b)


@gpu
def test_a_layer_can_be_captured_and_replayed():
    def step(x, logits, first, second, grad):
        y = layer_of_experts(x, logits, first, second, 2, False)
        return (y, *torch.autograd.grad(y, (x, logits, first, second), grad))

    arguments = arguments_of_a_layer(40, torch.float16)
    step(*arguments)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(*arguments)
    for turn in range(4):
        fresh = arguments_of_a_layer(50 + turn, torch.float16)
        with torch.no_grad():
            for a, f in zip(arguments, fresh):
                a.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(results, step(*fresh)):
            assert torch.equal(a, b), turn


def parts():
    """Name, a part of a model that begins with operators of torch and ends with one on tokens, and its arguments."""
    g = generator(60)
    leaf = lambda *s: normal(g, *s).requires_grad_()  # noqa: E731
    places = places_of(g, 30, 2)
    return [("route", lambda l: tokens.route(torch.tanh(l * 2), 3)[0], (leaf(30, 9),)),
            ("dispatch", lambda x: tokens.dispatch(torch.exp(x) * x, places), (leaf(30, 12),)),
            ("combine", lambda r, w, x: tokens.combine(torch.sigmoid(r), places, w.square(), torch.sin(x)), (leaf(60, 12), leaf(30, 2), leaf(30, 12)))]


@gpu
@pytest.mark.parametrize("which", range(3))
def test_backward_passes_as_autograd_runs_them(which):
    """Parts that a checkpoint runs again; saved tensors that come back on the host; gradients of gradients."""
    name, part, arguments = parts()[which]
    say(name)
    y = part(*arguments)
    grad = torch.cos(torch.arange(y.numel(), device="cuda", dtype=torch.float32)).view(y.shape)
    expected = torch.autograd.grad(y, arguments, grad)
    again = checkpoint(part, *arguments, use_reentrant=False)
    assert torch.equal(again, y)
    for a, e in zip(torch.autograd.grad(again, arguments, grad), expected):
        assert torch.equal(a, e)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        y = part(*(a.detach().requires_grad_() for a in arguments))
    node = y.grad_fn
    with pytest.raises(RuntimeError, match="another device"):
        node(grad)
    with pytest.raises(RuntimeError, match="GPU"):
        part(*arguments).grad_fn(grad.cpu())
    with torch.autograd.graph.save_on_cpu():
        away = part(*arguments)
    for a, e in zip(torch.autograd.grad(away, arguments, grad), expected):
        assert torch.equal(a, e)
    first, = torch.autograd.grad(part(*arguments).square().sum(), arguments[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated"):
        first.sum().backward()
    with torch.no_grad():
        assert not part(*arguments).requires_grad


@gpu
def test_an_index_that_was_changed_has_no_gradient():
    logits = torch.randn(8, 5, device="cuda", requires_grad=True)
    weights, index = tokens.route(logits, 2)
    index.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        weights.sum().backward()


@gpu
@pytest.mark.parametrize("weighted", [False, True])
def test_combine_keeps_only_what_its_gradients_read(weighted):
    """Rows are read for the weights' gradient, weights for the rows': what no wanted gradient reads may change, and is not held."""
    g = generator(8)
    places = places_of(g, 30, 2)
    place, token, has, _ = rows_reference(places, 5)
    values = {"rows": normal(g, 60, 5), "weights": normal(g, 30, 2) if weighted else None, "residual": normal(g, 30, 5)}
    dy = normal(g, 30, 5)
    flat = values["weights"].flatten()[has].double()[:, None] if weighted else 1.0
    drows, dweights, size = (torch.zeros(60, n, dtype=torch.float64, device="cuda") for n in (5, 1, 1))
    drows[place] = dy[token].double() * flat
    products = dy[token].double() * values["rows"][place].double()
    dweights[has], size[has] = products.sum(1, keepdim=True), products.abs().sum(1, keepdim=True)
    expected = {"rows": (drows, U * drows.abs()), "weights": (dweights.view(30, 2), 9 * U * size.view(30, 2)), "residual": (dy.double(), torch.zeros_like(dy))}
    reads = {"rows": {"weights"}, "weights": {"rows"}, "residual": set()}
    for wanted in ("rows", "weights", "residual")[::1 if weighted else 2]:
        for changed in ("rows", "weights", "residual")[::1 if weighted else 2]:
            given = {name: v.clone() if v is not None else None for name, v in values.items()}
            given[wanted].requires_grad_()
            y = tokens.combine(given["rows"], places, given["weights"], given["residual"])
            with torch.no_grad():
                given[changed].fill_(float("nan"))
            if changed in reads[wanted]:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(y, given[wanted], dy)
            else:
                near(torch.autograd.grad(y, given[wanted], dy)[0], *expected[wanted], wanted)
    rows = torch.zeros(60, 1 << 16, device="cuda")   # 16 MB
    residual = torch.zeros(30, 1 << 16, device="cuda", requires_grad=True)
    y = tokens.combine(rows, places, values["weights"], residual)
    held = torch.cuda.memory_allocated()
    del rows
    assert held - torch.cuda.memory_allocated() >= 60 << 18
    assert y.grad_fn is not None


@gpu
def test_no_kernel_is_compiled_late():
    """Calls of every kind of size find their kernels where qmlp.tokens.precompile left them."""
    g = generator(70)
    before = _lib.kernel_cache_stats()[0]
    for dtype in DTYPES:
        for experts in (3, 40, 100, 200, 500, 900, 2000):
            logits = normal(g, 9, experts, dtype=dtype).requires_grad_()
            weights, index = tokens.route(logits, 2)
            weights.sum().backward()
        places = tokens.group(index, 2000, places=True)[2]
        for channels in (1, 5, 20, 70, 150, 300, 600, 3000):
            x = normal(g, 9, channels, dtype=dtype).requires_grad_()
            tokens.combine(tokens.dispatch(x, places), places, weights.detach().requires_grad_(), x).sum().backward()
    assert _lib.kernel_cache_stats()[0] == before


@gpu
def test_example_serves_numbers_of_four_bits():
    """Trained for a few steps, then with the experts' weights in 4 bits: it runs, and refuses to be trained."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_experts.py")
    spec = importlib.util.spec_from_file_location("token_experts", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    torch.manual_seed(1)
    shapes = module.balls(20)
    model = module.ObjectFields(20)
    module.fit(model, *shapes, 3, batch=8, points=16)
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in model.experts.parameters())
    x = torch.randn(30, 32, device="cuda")
    layer = model.experts
    weights = [tokens.quantise_mx4(l.weight.detach()).dequantise() for l in (layer.first, layer.second)]
    layer.quantise()
    with torch.no_grad():
        assert bool(layer(x).isfinite().all())
        index, positions, _ = module.batch_of(*shapes, 8, 16)
        assert bool(model(index, positions).isfinite().all())
        for l, w in zip((layer.first, layer.second), weights):
            assert torch.equal(tokens.Mx4(l.codes, l.scales, l.inputs).dequantise(), w)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(x)


# ------------------------------------------------------------------------------------------------ refusals
@gpu
def test_arguments_that_do_not_fit_are_refused():
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
    for call, match in [
            (lambda: tokens.route(f(3, 4), 5), "no more than there are"),
            (lambda: tokens.route(f(3, 4), 0), "between 1 and 64"),
            (lambda: tokens.route(f(3, 100), 65), "between 1 and 64"),
            (lambda: tokens.route(f(3, 4, dtype=torch.float64), 2), "float, half or bfloat16"),
            (lambda: tokens.dispatch(f(3, 4), i32(4, 2)), "those of the tokens"),
            (lambda: tokens.dispatch(f(3, 4), i32(3)), "dimensions"),
            (lambda: tokens.dispatch(f(3, 4), i32(3, 0)), "at least one"),
            (lambda: tokens.dispatch(f(3, 4), i32(3, 2).long()), "INT32"),
            (lambda: tokens.dispatch(f(3, 4, dtype=torch.float64), i32(3, 2)), "float, half or bfloat16"),
            (lambda: tokens.combine(f(5, 4), i32(3, 2)), "must have 6 entries"),
            (lambda: tokens.combine(f(6, 4), i32(3, 2), f(3, 3)), "shape of places"),
            (lambda: tokens.combine(f(6, 4), i32(3, 2), f(3, 2, dtype=torch.float16)), "rows' type or FLOAT"),
            (lambda: tokens.combine(f(6, 4), i32(3, 2), None, f(3, 5)), "residual"),
            (lambda: tokens.combine(f(6, 4), i32(3, 2), None, f(3, 4, dtype=torch.float16)), "must be of type FLOAT"),
            (lambda: tokens.combine(f(6), i32(3, 2)), "2 dimensions")]:
        with pytest.raises((qmlp.QmlpError, RuntimeError, ValueError, TypeError), match=match):
            call()


@gpu
def test_function_transforms_and_tangents_are_refused():
    x, places = torch.randn(2, 3, 4, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2)
    for call, v in ((lambda v: tokens.route(v, 2)[0], x), (lambda v: tokens.dispatch(v, places), x),
                    (lambda v: tokens.combine(v, places), torch.randn(2, 6, 4, device="cuda"))):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(v)
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: call(t).sum())(v[0])
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(torch.autograd.forward_ad.make_dual(v[0], torch.ones_like(v[0])))
        call(v[0])


def test_tensors_on_the_host_are_refused():
    places = torch.zeros(3, 2, dtype=torch.int32)
    for call in (lambda: tokens.route(torch.zeros(3, 4), 2), lambda: tokens.dispatch(torch.zeros(3, 4), places),
                 lambda: tokens.combine(torch.zeros(6, 4), places)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_c_interface_refuses_before_any_launch():
    """Descriptors that do not fit end in a status and a message; nothing of them is read (these calls need no device)."""
    lib, F, H, I = _lib.lib, _lib.QMLP_FLOAT, _lib.QMLP_HALF, _lib.QMLP_INT32
    none = _lib.TensorDesc()
    logits, weights, index = descriptor(F, 4, 6), descriptor(F, 4, 2), descriptor(I, 4, 2)
    route = lambda l, w, i: lib.qmlp_tokens_route(l, 0, w, i, None)  # noqa: E731
    refused(route(descriptor(F, 4, 6, strides=(12, 2)), weights, index), "consecutive")
    refused(route(logits, descriptor(H, 4, 2), index), "must be of type FLOAT")
    refused(route(logits, weights, descriptor(F, 4, 2)), "must be of type INT32")
    refused(route(logits, descriptor(F, 4, 3), index), "must have 2 entries")
    refused(route(logits, descriptor(F, 4, 7), descriptor(I, 4, 7)), "no more than there are")
    refused(route(descriptor(F, 4, 70), descriptor(F, 4, 65), descriptor(I, 4, 65)), "between 1 and 64")
    refused(route(logits, descriptor(F, 4, 2, strides=(1, 1)), index), "share memory")
    refused(route(logits, weights, descriptor(I, 4, 2, strides=(0, 1))), "share memory")
    refused(route(none, weights, index), "undefined")
    many = 2 ** 31 - 2 ** 12 + 1
    refused(route(descriptor(H, 1, many), descriptor(H, 1, 2), descriptor(I, 1, 2)), "experts must not be more")
    refused(lib.qmlp_tokens_route_adjoint(logits, index, weights, 0, descriptor(F, 4, 5), None), "must have 6 entries")
    refused(lib.qmlp_tokens_route_adjoint(logits, index, descriptor(F, 3, 2), 0, logits, None), "must have 4 entries")
    x, places, rows = descriptor(F, 4, 6), descriptor(I, 4, 2), descriptor(F, 8, 6)
    refused(lib.qmlp_tokens_dispatch(x, places, descriptor(F, 7, 6), None), "must have 8 entries")
    refused(lib.qmlp_tokens_dispatch(descriptor(F, 4, 5), places, rows, None), "must have 6 entries")
    refused(lib.qmlp_tokens_dispatch(descriptor(H, 4, 6), places, rows, None), "must be of type FLOAT")
    refused(lib.qmlp_tokens_dispatch(x, descriptor(F, 4, 2), rows, None), "must be of type INT32")
    refused(lib.qmlp_tokens_dispatch(x, places, descriptor(F, 8, 6, strides=(3, 1)), None), "share memory")
    refused(lib.qmlp_tokens_dispatch(descriptor(F, 1 << 30, 6, strides=(0, 1)), descriptor(I, 1 << 30, 2), rows, None), "fit into 32 bits")
    refused(lib.qmlp_tokens_dispatch(descriptor(H, 1, many), descriptor(I, 1, 1), descriptor(H, 1, many), None), "channels must not be more")
    refused(lib.qmlp_tokens_combine(rows, places, descriptor(H, 4, 2), none, x, None), "rows' type or FLOAT")
    refused(lib.qmlp_tokens_combine(rows, places, descriptor(F, 4, 3), none, x, None), "must have 2 entries")
    refused(lib.qmlp_tokens_combine(rows, places, none, descriptor(F, 4, 5), x, None), "must have 6 entries")
    refused(lib.qmlp_tokens_combine(rows, places, none, none, descriptor(F, 4, 6, strides=(0, 1)), None), "share memory")
    refused(lib.qmlp_tokens_combine_adjoint(rows, places, none, x, descriptor(F, 8, 5), none, None), "must have 6 entries")
    refused(lib.qmlp_tokens_combine_adjoint(descriptor(H, 8, 6), places, descriptor(H, 4, 2), descriptor(H, 4, 6), none, descriptor(F, 4, 2), None),
            "must be of type HALF")
    order, offsets = descriptor(I, 8), descriptor(I, 4)
    refused(lib.qmlp_tokens_group_places(descriptor(I, 8), 3, order, offsets, descriptor(I, 7), None, None), "must have 8 entries")
    refused(lib.qmlp_tokens_group_places(descriptor(I, 8), 3, order, offsets, descriptor(F, 8), None, None), "must be of type INT32")


def test_gradients_of_combine_refuse_missing_rows():
    """Rows are needed for the weights' gradient; without it the rows' gradient has the sizes (these calls need no device)."""
    lib, F, I = _lib.lib, _lib.QMLP_FLOAT, _lib.QMLP_INT32
    none, places, dy, drows, w = _lib.TensorDesc(), descriptor(I, 4, 2), descriptor(F, 4, 6), descriptor(F, 8, 6), descriptor(F, 4, 2)
    adjoint = lambda *a: lib.qmlp_tokens_combine_adjoint(*a, None)  # noqa: E731
    refused(adjoint(none, places, w, dy, drows, w), "rows is undefined")
    refused(adjoint(none, places, w, dy, none, none), "rows is undefined")
    refused(adjoint(none, places, w, dy, descriptor(F, 7, 6), none), "must have 8 entries")
    refused(adjoint(none, places, w, descriptor(F, 4, 5), drows, none), "must have 6 entries")
    refused(adjoint(none, places, descriptor(_lib.QMLP_HALF, 4, 2), dy, drows, none), "rows' type or FLOAT")
    refused(adjoint(none, places, none, dy, descriptor(F, 8, 6, strides=(3, 1)), none), "share memory")
