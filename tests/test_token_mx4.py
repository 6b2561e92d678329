"""Numbers of 4 bits and the experts' layers with them (qmlp.tokens) against their definitions in 64 bits.

Codes, scales and the values that they stand for are exact. Sums of n products in 32 bits are off by at most n 2^-23 of the sum of their magnitudes, a
result is rounded once to its type.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import qmlp
from qmlp import _lib, tokens
from token_helpers import DTYPES, U, Margins, described, descriptor, generator, near, normal, offsets_of, refused, say, skip_warming

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_warming(request):
    skip_warming(request)


VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantised_reference(x):
    """Codes (one a number) and biased exponents of rows, from the definition."""
    x = x.double().cpu().numpy()
    rows, columns = x.shape
    blocks = -(-columns // 32)
    padded = np.zeros((rows, blocks * 32))
    padded[:, :columns] = x
    padded = padded.reshape(rows, blocks, 32)
    largest = np.abs(padded).max(2)
    bad = ~np.isfinite(largest)
    with np.errstate(divide="ignore", invalid="ignore"):
        exponent = np.where(largest > 0, np.frexp(np.where(bad, 1.0, largest))[1] - 1 - 2, -127)
    exponent = np.clip(exponent, -127, 127)
    v = np.where(bad[..., None], 0.0, padded) / np.exp2(exponent)[..., None]
    distance = np.abs(np.abs(v)[..., None] - VALUES)
    # the nearest; of two the one whose code is even
    code = np.argmin(distance, 3)
    tie = np.take_along_axis(distance, np.minimum(code + 1, 7)[..., None], 3)[..., 0] == np.take_along_axis(distance, code[..., None], 3)[..., 0]
    code = np.where(tie & (code % 2 == 1) & (code < 7), code + 1, code)
    code = np.where(bad[..., None], 0, code + 8 * (np.signbit(v) & ~bad[..., None]))
    return code.reshape(rows, -1), np.where(bad, 255, exponent + 127)


def values_reference(code, scale, columns):
    v = np.where(code >= 8, -1.0, 1.0) * VALUES[code % 8]
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    return torch.from_numpy((v.reshape(*scale.shape, 32) * s[..., None]).reshape(v.shape)[:, :columns])


def unpacked(codes):
    c = codes.cpu().numpy()
    return np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)


def check(x, what):
    q = tokens.quantise_mx4(x)
    code, scale = quantised_reference(x)
    assert q.codes.dtype == q.scales.dtype == torch.uint8 and q.shape == x.shape
    assert np.array_equal(q.scales.cpu().numpy(), scale), what
    assert np.array_equal(unpacked(q.codes), code), what
    exact = values_reference(code, scale, x.shape[1])
    for dtype in DTYPES:
        values = q.dequantise(dtype)
        assert values.dtype == dtype and values.shape == x.shape
        expected = exact.to(dtype)   # (one rounding; float32 and bfloat16 need none)
        assert torch.equal(values.cpu().nan_to_num(7.0, posinf=8.0, neginf=9.0), expected.nan_to_num(7.0, posinf=8.0, neginf=9.0)), (what, dtype)
        assert torch.equal(values.cpu().isnan(), expected.isnan())
    return q


# ------------------------------------------------------------------------------------------------ numbers
@gpu
@pytest.mark.parametrize("columns", [1, 7, 8, 31, 32, 33, 40, 63, 64, 65, 100, 333, 512, 777, 2048])
@pytest.mark.parametrize("rows", [1, 3, 200])
@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_of_four_bits(rows, columns, dtype):
    say("numbers", rows, columns, dtype)
    g = generator(columns + rows)
    check((normal(g, rows, columns) * torch.exp(3 * normal(g, columns))).to(dtype), "random")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_number_and_what_lies_between(dtype):
    """Halfway between two numbers, beside it, beyond the largest, signed zeros; at many scales."""
    eps = torch.finfo(dtype).eps
    points = [s * v * (1 + d) for v in (0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.5) for d in (-eps, 0, eps) for s in (1, -1)]
    points += [0.0, -0.0] + [7.9, -7.9] * 2
    exponents = range(-14, 13) if dtype == torch.float16 else range(-126, 125, 7)
    rows = []
    for e in exponents:
        for at in range(0, len(points), 31):
            rows.append([4.0 * 2.0 ** e] + [math.ldexp(p, e) for p in (points[at:at + 31] + [0.0] * 31)[:31]])
    check(torch.tensor(rows, dtype=torch.float64).to(dtype).cuda(), "points")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_largest_smallest_and_empty_blocks(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(12, 40, dtype=dtype, device="cuda")
    x[1] = info.max
    x[2, ::2], x[2, 1] = -info.max, info.tiny
    x[3] = info.smallest_normal
    x[4] = -info.smallest_normal * info.eps       # the smallest number of all
    x[5, 3], x[5, 4] = info.smallest_normal, info.max
    x[6, 0] = info.smallest_normal * info.eps
    x[7, 33] = 1.0
    x[8] = -0.0
    check(x, "extremes")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_a_number_stays_in_its_block(dtype):
    g = generator(4)
    x = normal(g, 6, 100, dtype=dtype)
    x[1, 40], x[2, 99], x[3, 0], x[4, 64:] = float("nan"), float("inf"), -float("inf"), -float("nan")
    q = check(x, "not numbers")
    assert (q.scales == 255).sum(1).tolist() == [0, 1, 1, 1, 2, 0]


@gpu
def test_numbers_of_other_shapes_and_strides():
    g = generator(5)
    wide = normal(g, 5, 6, 90)
    for x in (wide[..., 3:70], wide.transpose(0, 1)[..., :33], wide[..., ::2], wide[:1].expand(5, 6, 90), wide[0, 0], wide[:0]):
        q = tokens.quantise_mx4(x)
        flat = x.reshape(-1, x.shape[-1]).contiguous()
        p = tokens.quantise_mx4(flat)
        assert q.shape == x.shape
        assert torch.equal(q.codes.reshape(p.codes.shape), p.codes) and torch.equal(q.scales.reshape(p.scales.shape), p.scales)
        assert torch.equal(q.dequantise().reshape(flat.shape), p.dequantise())
    some = tokens.quantise_mx4(wide.reshape(30, 90))
    part = tokens.Mx4(some.codes[3:20:2, 16:], some.scales[3:20:2, 1:], 58)
    assert torch.equal(part.dequantise(), some.dequantise()[3:20:2, 32:])


@gpu
def test_more_than_two_to_the_31_numbers():
    rows, columns = (1 << 20) + 5, 2080
    x = torch.zeros(rows, columns, dtype=torch.bfloat16, device="cuda")
    x[-1], x[-2, 2079] = 3.0, 96.0
    q = tokens.quantise_mx4(x)
    assert int(torch.count_nonzero(q.codes)) == 2080 // 2 + 1 and q.scales[-1].tolist() == [126] * 65 and int(q.scales[-2, 64]) == 127 + 4
    assert torch.equal(q.dequantise(torch.bfloat16)[-3:], x[-3:])


# ------------------------------------------------------------------------------------------------ layers
COUNTS = {
    "one row": [1],
    "one row of many experts": [0, 0, 1, 0] + [0] * 70,
    "nothing": [0, 0, 0],
    "ragged": [5, 0, 130, 1, 64, 0, 0, 257, 33],
    "one has all": [0, 0, 3000, 0],
    "hundreds of experts": [(7 * i) % 13 for i in range(300)],
    "many rows": [5000, 4097, 1],
}


def linear_reference(x, weight, counts, bias):
    y, error = (torch.zeros(x.shape[0], weight.shape[1], dtype=torch.float64, device=x.device) for _ in range(2))
    at = 0
    for e, n in enumerate(counts):
        p = slice(at, at + n)
        at += n
        y[p] = x[p] @ weight[e].T + (bias[e].double() if bias is not None else 0)
        error[p] = (x.shape[1] + 8) * U * (x[p].abs() @ weight[e].abs().T + (bias[e].double().abs() if bias is not None else 0))
    return y, error


def check_linear(counts, inputs, outputs, dtype, seed, ungrouped=0, biased=True):
    g = generator(seed)
    rows = sum(counts) + ungrouped
    x, weight = normal(g, rows, inputs, dtype=dtype), tokens.quantise_mx4(normal(g, len(counts), outputs, inputs) * torch.exp(normal(g, inputs)))
    bias = normal(g, len(counts), outputs, dtype=dtype) if biased else None
    y = tokens.mx4_linear(x, weight, offsets_of(counts), bias)
    q = tokens.quantise_mx4(x)
    exact, error = linear_reference(q.dequantise().double(), weight.dequantise().double(), counts, bias)
    assert y.dtype == dtype
    near(y, exact, error, "y")
    near(tokens.mx4_linear(q, weight, offsets_of(counts), bias, dtype), exact, error, "y of codes")   # (which may be added up in another order)
    assert torch.equal(tokens.mx4_linear(x, weight, offsets_of(counts), bias), y)


@gpu
@pytest.mark.parametrize("counts", list(COUNTS))
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (3, 5), (32, 16), (64, 64), (64, 56), (77, 130), (200, 33), (256, 512), (1030, 70)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_of_four_bits(counts, inputs, outputs, dtype):
    say("layers", counts, inputs, outputs, dtype)
    check_linear(COUNTS[counts], inputs, outputs, dtype, inputs + len(COUNTS[counts]), outputs % 7, inputs % 2 == 1)


@gpu
@pytest.mark.parametrize("inputs,outputs", [(2000, 40), (40, 2000), (1023, 1100), (4096, 16), (2048, 513)])
@pytest.mark.parametrize("counts", [[1], [3, 0, 9], [16], [17, 0, 32], [70, 0, 0, 31]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_of_few_rows(inputs, outputs, counts, dtype):
    say("few rows", inputs, outputs, counts, dtype)
    check_linear(counts, inputs, outputs, dtype, inputs, 2)


@gpu
@pytest.mark.parametrize("inputs,outputs", [(520, 264), (1024, 640), (96, 136), (2100, 300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_of_many_rows(inputs, outputs, dtype):
    """Enough work for larger tiles; experts whose rows end anywhere in one."""
    say("many rows", inputs, outputs, dtype)
    counts = [450 + (37 * e) % 140 for e in range(60)]
    counts[7], counts[20], counts[59] = 0, 1, 3000
    check_linear(counts, inputs, outputs, dtype, outputs, 5)


@gpu
@pytest.mark.parametrize("inputs", [1, 40, 256, 257, 500, 512, 520, 768, 1030, 1536, 2100])
@pytest.mark.parametrize("outputs", [1300, 1301])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layers_of_the_largest_tiles(inputs, outputs, dtype):
    """One tile of K and part of one, an odd and an even number of them; rows and outputs that end anywhere in one."""
    say("largest tiles", inputs, outputs, dtype)
    counts = [450 + (37 * e) % 140 for e in range(60)]
    counts[7], counts[20], counts[59] = 0, 1, 3000
    check_linear(counts, inputs, outputs, dtype, inputs + outputs, 5)


@gpu
@pytest.mark.parametrize("experts", [63, 64, 65, 128, 511, 513, 4096, 4097])
def test_numbers_of_experts(experts):
    say("numbers of experts", experts)
    check_linear([(11 * e + experts) % 5 * (e % 3 != 1) + 70 * (e in (0, 63, 64, experts - 1)) for e in range(experts)], 40, 8, torch.float16, experts, 3)


@gpu
@pytest.mark.parametrize("rows,outputs", [(5, 40), (70, 40), (3000, 300), (33000, 1030)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_expert_are_zeros(rows, outputs, dtype):
    """Without any expert, and behind the last one's rows: no weights are read for them."""
    weight = tokens.Mx4(torch.zeros(0, outputs, 32, dtype=torch.uint8, device="cuda"), torch.zeros(0, outputs, 2, dtype=torch.uint8, device="cuda"), 60)
    x = torch.ones(rows, 60, dtype=dtype, device="cuda")
    assert not bool(tokens.mx4_linear(x, weight, offsets_of([])).any())
    weight = tokens.Mx4(torch.full((2, outputs, 32), 0x22, dtype=torch.uint8, device="cuda"), torch.full((2, outputs, 2), 127, dtype=torch.uint8, device="cuda"), 60)
    bias = torch.ones(2, outputs, dtype=dtype, device="cuda")
    y = tokens.mx4_linear(x, weight, offsets_of([0, rows // 3]), bias)
    assert bool((y[:rows // 3] == 61).all()) and not bool(y[rows // 3:].any())


@gpu
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 300, 3000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_layer_needs_no_offsets(rows, dtype):
    g = generator(rows)
    x, weight = normal(g, rows, 300, dtype=dtype), tokens.quantise_mx4(normal(g, 1, 129, 300))
    y = tokens.mx4_linear(x, weight)
    assert torch.equal(y, tokens.mx4_linear(x, weight, offsets_of([rows])))
    exact, error = linear_reference(tokens.quantise_mx4(x).dequantise().double(), weight.dequantise().double(), [rows], None)
    near(y, exact, error, "y")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[37, 70, 5], [370, 700, 50], [3, 9, 1]])
def test_infinite_rows_of_one_expert_stay_with_it(dtype, counts):
    """An infinity makes its block NaN, and so the results of its row, no others; a block of NaN in the weights makes its output NaN."""
    g = generator(12)
    rows, first = sum(counts) + 8, counts[0]
    last = first + counts[1] - 1
    x, weight = normal(g, rows, 96, dtype=dtype), tokens.quantise_mx4(normal(g, 3, 40, 96))
    expected = tokens.mx4_linear(x, weight, offsets_of(counts))
    bad = x.clone()
    bad[first], bad[last, 50], bad[sum(counts):] = float("nan"), float("inf"), float("nan")
    y = tokens.mx4_linear(bad, weight, offsets_of(counts))
    keep = [r for r in range(rows) if r not in (first, last)]
    assert torch.equal(y[keep], expected[keep]) and bool(y[[first, last]].isnan().all())
    weight.scales[1, 7, 2] = 255
    y = tokens.mx4_linear(x, weight, offsets_of(counts))
    assert bool(y[first:last + 1, 7].isnan().all())
    expected[first:last + 1, 7] = 0
    y[first:last + 1, 7] = 0
    assert torch.equal(y, expected)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layers_of_other_strides(dtype):
    """Rows and matrices that lie apart, begin at odd addresses, or are one and the same."""
    g = generator(14)
    counts = [70, 0, 200, 31]
    wide = normal(g, 310, 200, dtype=dtype)
    stack = tokens.quantise_mx4(normal(g, 8, 90, 192))
    for x in (wide[:, 1:65], wide[:, 3:67], wide[5:, :64], wide.t()[:200].t()[:, :64]):
        x = x[:301]
        for part in (slice(0, 4), slice(1, 8, 2)):
            for block in (0, 1, 3):
                codes, scales = stack.codes[part, 5:72, 16 * block:16 * block + 32], stack.scales[part, 5:72, block:block + 2]
                weight = tokens.Mx4(codes, scales, 64)
                packed = tokens.Mx4(codes.contiguous(), scales.contiguous(), 64)
                y = tokens.mx4_linear(x, weight, offsets_of(counts))
                exact, error = linear_reference(tokens.quantise_mx4(x).dequantise().double(), packed.dequantise().double(), counts, None)
            near(y, exact, error, "y")
        shared = tokens.Mx4(stack.codes[:1, :, :32].expand(4, 90, 32), stack.scales[:1, :, :2].expand(4, 90, 2), 64)
        y = tokens.mx4_linear(x, shared, offsets_of(counts))
        first = tokens.Mx4(stack.codes[:1, :, :32], stack.scales[:1, :, :2], 64)
        exact, error = linear_reference(tokens.quantise_mx4(x).dequantise().double(), first.dequantise().double(), [301], None)
        near(y, exact, error, "y")
    odd = torch.zeros(90 * 32 + 1, dtype=torch.uint8, device="cuda")
    codes = odd[1:].view(1, 90, 32)
    codes.copy_(stack.codes[:1, :, :32])
    x = wide[:, :64]
    first = tokens.Mx4(stack.codes[:1, :, :32], stack.scales[:1, :, :2], 64)
    exact, error = linear_reference(tokens.quantise_mx4(x).dequantise().double(), first.dequantise().double(), [310], None)
    near(tokens.mx4_linear(x, tokens.Mx4(codes, stack.scales[:1, :, :2], 64)), exact, error, "y")


@gpu
@pytest.mark.parametrize("block", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weights_that_begin_at_any_block_of_others(block, dtype):
    """Parts of wider matrices of codes, whose scales then begin at any byte, of all experts or of every other one."""
    g = generator(15 + block)
    counts = [70, 0, 200, 31]
    wide = normal(g, 310, 200, dtype=dtype)
    stack = tokens.quantise_mx4(normal(g, 8, 90, 192))
    for x in (wide[:, 1:65], wide[5:, :64]):
        x = x[:301]
        for part in (slice(0, 4), slice(1, 8, 2)):
            weight = tokens.Mx4(stack.codes[part, 5:72, 16 * block:16 * block + 32], stack.scales[part, 5:72, block:block + 2], 64)
            packed = tokens.Mx4(weight.codes.contiguous(), weight.scales.contiguous(), 64)
            exact, error = linear_reference(tokens.quantise_mx4(x).dequantise().double(), packed.dequantise().double(), counts, None)
            near(tokens.mx4_linear(x, weight, offsets_of(counts)), exact, error, "y")


@gpu
@pytest.mark.parametrize("counts,outputs", [([2, 1], 40), ([37, 70, 0, 5], 72), ([900, 0, 2101], 300)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_codes_of_other_strides(counts, outputs, dtype):
    """Rows that are numbers of 4 bits already: parts of wider ones, every other one, one and the same, codes at odd addresses."""
    say("codes of rows", counts, outputs, dtype)
    g = generator(16 + outputs)
    rows = sum(counts) + 3
    stack, weight = tokens.quantise_mx4(normal(g, 2 * rows + 4, 700)), tokens.quantise_mx4(normal(g, len(counts), outputs, 600))
    bias = normal(g, len(counts), outputs, dtype=dtype)
    odd = torch.zeros(rows * 19 * 16 + 1, dtype=torch.uint8, device="cuda")[1:].view(rows, 19 * 16)
    odd.copy_(stack.codes[:rows, :19 * 16])
    odd_row = torch.zeros(rows, 19 * 16 + 8, dtype=torch.uint8, device="cuda")[:, :19 * 16]
    odd_row.copy_(stack.codes[:rows, :19 * 16])
    one = lambda t: t[3:4].expand(rows, t.shape[1])  # noqa: E731
    # (codes of 600 of the 700 columns: the last 8 numbers of block 18 meet weights that are zeros)
    for codes, scales in ((stack.codes[1:rows + 1, :19 * 16], stack.scales[1:rows + 1, :19]), (stack.codes[3:2 * rows + 3:2, 16:20 * 16], stack.scales[3:2 * rows + 3:2, 1:20]),
                          (odd, stack.scales[:rows, :19]), (odd_row, stack.scales[:rows, :19]), (one(stack.codes[:, :19 * 16]), one(stack.scales[:, :19]))):
        values = tokens.Mx4(codes.contiguous(), scales.contiguous(), 600).dequantise().double()
        exact, error = linear_reference(values, weight.dequantise().double(), counts, bias)
        near(tokens.mx4_linear(tokens.Mx4(codes, scales, 600), weight, offsets_of(counts), bias, dtype), exact, error, "y")


@gpu
@pytest.mark.parametrize("inputs", [40, 700])
@pytest.mark.parametrize("experts", [65, 128, 513, 4096, 4097])
def test_more_experts_than_rows(experts, inputs):
    """Tiles begin at the first rows of experts, which are found among all of them: the first, the last, some in between, of more than a tile."""
    say("experts", experts, inputs)
    counts = [0] * experts
    for e, n in ((0, 3), (1, 1), (experts // 2, 17), (experts // 2 + 1, 2), (experts - 2, 1), (experts - 1, 20)):
        counts[e] += n
    for dtype in (torch.float32, torch.bfloat16):
        check_linear(counts, inputs, 24, dtype, experts + inputs, 3)
    counts[0], counts[experts - 1], counts[63] = 0, 0, 16
    check_linear(counts, inputs, 24, torch.float16, experts + inputs, 0, False)


@gpu
@pytest.mark.parametrize("offsets", [[0, 50, 1 << 30, 1 << 30, 1 << 30], [0, -5, -7, 1000, 20], [90, 80, 70, 60, 50], [2 ** 31 - 1] * 5, [-2 ** 31] * 5,
                                     [0, 33, 33, 64, 97]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,inputs,outputs", [(97, 16, 24), (97, 2001, 33), (2100, 64, 72)])
def test_nothing_beside_the_results_is_written(offsets, dtype, rows, inputs, outputs):
    """Offsets that make no sense give no sensible rows, but what the calls write is within their results and their memory."""
    say("beside", offsets, dtype, rows, inputs, outputs)
    lib, size, none = _lib.lib, ctypes.c_size_t(), _lib.TensorDesc()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    blocks = (inputs + 31) // 32
    margins = Margins()
    x, w = torch.ones(rows, inputs, dtype=dtype, device="cuda"), torch.ones(4 * outputs, inputs, device="cuda")
    codes, scales = margins.tensor(torch.uint8, 4 * outputs, 16 * blocks), margins.tensor(torch.uint8, 4 * outputs, blocks)
    _lib.check(lib.qmlp_tokens_mx4_quantise(described(w), described(codes), described(scales), stream))
    values, y = margins.tensor(dtype, 4 * outputs, inputs), margins.tensor(dtype, rows, outputs)
    _lib.check(lib.qmlp_tokens_mx4_values(described(codes), described(scales), described(values), stream))
    _lib.check(lib.qmlp_tokens_mx4_linear_memory(rows, 4, inputs, outputs, ctypes.byref(size)))
    memory = margins.bytes(size.value)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    _lib.check(lib.qmlp_tokens_mx4_linear(described(x), none, described(codes.view(4, outputs, -1)), described(scales.view(4, outputs, -1)), described(off), none,
                                          described(y), memory, stream))
    torch.cuda.synchronize()
    margins.untouched()
    assert bool((values == 1).all())


# ------------------------------------------------------------------------------------------------ together
def served_layer(x, logits, first, second, chosen):
    """Router, sort, rows to the experts, their layers of 4 bits, and back on top of the tokens."""
    weights, index = tokens.route(logits, chosen, True)
    _, offsets, places = tokens.group(index, first.codes.shape[0], places=True)
    rows = torch.relu(first(tokens.dispatch(x, places), offsets))
    return tokens.combine(second(rows, offsets), places, weights, x)


def layers(seed, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    pair = [qmlp.FusedGroupedLinear(8, *s, dtype=dtype) for s in ((96, 200), (200, 96))]
    for l in pair:
        l.bias.data.normal_(0, 0.1)
    return [tokens.FusedMx4GroupedLinear(l) for l in pair]


@gpu
@pytest.mark.parametrize("rows", [1, 24, 900])
def test_a_served_layer_of_experts(rows):
    """From one token on; the layers' weights of 4 bits as they are, rows rounded where the calls round them."""
    g = generator(rows)
    first, second = layers(1)
    x, logits = normal(g, rows, 96, dtype=torch.bfloat16), normal(g, rows, 8, dtype=torch.bfloat16)
    y = served_layer(x, logits, first, second, 2)
    # the same one call after the other, every result checked with what the call was given
    weights, index = tokens.route(logits, 2, True)
    _, offsets, places = tokens.group(index, 8, places=True)
    counts = offsets.diff().tolist()
    r = tokens.dispatch(x, places)
    for layer in (first, second):
        out = layer(r, offsets)
        numbers = tokens.Mx4(layer.codes, layer.scales, layer.inputs).dequantise().double()
        exact, error = linear_reference(tokens.quantise_mx4(r).dequantise().double(), numbers, counts, layer.bias)
        near(out, exact, error, "layer")
        r = torch.relu(out) if layer is first else out
    exact, size = x.double(), x.double().abs()
    for j in range(2):
        term = weights[:, j:j + 1].double() * r.double()[places[:, j].long()]
        exact, size = exact + term, size + term.abs()
    near(y, exact, 4 * U * size, "combined")


@gpu
def test_calls_run_on_the_current_stream_and_can_be_captured():
    first, second = layers(2)
    arguments = lambda seed: (lambda g: [normal(g, 50, 96, dtype=torch.bfloat16), normal(g, 50, 8, dtype=torch.bfloat16)])(generator(seed))  # noqa: E731
    expected = served_layer(*arguments(1), first, second, 2)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = served_layer(*arguments(1), first, second, 2)
    stream.synchronize()
    assert torch.equal(late, expected)
    held = arguments(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = served_layer(*held, first, second, 2)
        numbers = tokens.quantise_mx4(held[0])
        values = numbers.dequantise()
    for turn in range(4):
        fresh = arguments(10 + turn)
        for a, f in zip(held, fresh):
            a.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(results, served_layer(*fresh, first, second, 2)), turn
        assert torch.equal(values, tokens.quantise_mx4(fresh[0]).dequantise()), turn


@gpu
def test_no_kernel_is_compiled_late():
    """Calls of every kind of size find their kernels where qmlp.tokens.precompile left them."""
    g = generator(71)
    before = _lib.kernel_cache_stats()[0]
    for dtype in DTYPES:
        for rows, experts, inputs, outputs in ((4, 8, 100, 100), (4, 1, 4096, 64), (16, 1, 4096, 512), (1, 300, 64, 1024), (300, 2, 64, 64), (9000, 2, 64, 256),
                                               (33000, 2, 64, 1030)):
            x, weight = normal(g, rows, inputs, dtype=dtype), tokens.quantise_mx4(normal(g, experts, outputs, inputs))
            offsets = offsets_of([rows] + [0] * (experts - 1))
            for values in (x, tokens.quantise_mx4(x)):
                tokens.mx4_linear(values, weight, offsets, None, dtype)
            tokens.quantise_mx4(x).dequantise(dtype)
    assert _lib.kernel_cache_stats()[0] == before


@gpu
def test_module_keeps_its_numbers():
    first, _ = layers(3)
    state = first.state_dict()
    assert sorted(state) == ["bias", "codes", "scales"] and not list(first.parameters())
    other, _ = layers(4)
    other.load_state_dict(state)
    x = torch.randn(9, 96, device="cuda")
    offsets = offsets_of([1, 2, 3, 0, 0, 0, 2, 1])
    assert torch.equal(first(x, offsets), other(x, offsets)) and first(x, offsets).dtype == torch.float32


# ------------------------------------------------------------------------------------------------ refusals
@gpu
def test_arguments_that_do_not_fit_are_refused():
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    i32 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)  # noqa: E731
    weight = tokens.quantise_mx4(f(2, 5, 40))
    for call, match in [
            (lambda: tokens.quantise_mx4(f(3, 4, dtype=torch.float64)), "float, half or bfloat16"),
            (lambda: tokens.quantise_mx4(f(3, 4).requires_grad_()), "no gradient"),
            (lambda: weight.dequantise(torch.float64), "float, half or bfloat16"),
            (lambda: tokens.Mx4(weight.codes, weight.scales, 65), "blocks"),
            (lambda: tokens.Mx4(weight.codes[..., :16], weight.scales, 40), "blocks"),
            (lambda: tokens.mx4_linear(f(3, 41), weight, i32(3)), "inputs"),
            (lambda: tokens.mx4_linear(f(3, 40), weight), "one expert"),
            (lambda: tokens.mx4_linear(f(3, 40), weight, i32(2)), "must have 3 entries"),
            (lambda: tokens.mx4_linear(f(3, 40), weight, i32(3).long()), "INT32"),
            (lambda: tokens.mx4_linear(f(3, 40), weight, i32(3), f(2, 4)), "must have 5 entries"),
            (lambda: tokens.mx4_linear(f(3, 40), weight, i32(3), f(2, 5, dtype=torch.float16)), "must be of type FLOAT"),
            (lambda: tokens.mx4_linear(f(3, 40).requires_grad_(), weight, i32(3)), "no gradient"),
            (lambda: tokens.mx4_linear(f(3, 40), weight, i32(3), f(2, 5).requires_grad_()), "no gradient"),
            (lambda: tokens.mx4_linear(tokens.quantise_mx4(f(3, 40)), weight, i32(3), None, torch.float64), "float, half or bfloat16"),
            (lambda: tokens.mx4_linear(tokens.quantise_mx4(f(3, 40)), weight, i32(3), None, "bfloat16"), "dtype"),
            (lambda: tokens.mx4_linear(f(3, 40, dtype=torch.float64), weight, i32(3)), "float, half or bfloat16"),
            (lambda: tokens.mx4_linear(f(3, 4, 40), weight, i32(3)), "2 dimensions"),
            (lambda: tokens.mx4_linear(f(3, 40), tokens.quantise_mx4(f(5, 40)), i32(3)), "3 dimensions")]:
        with pytest.raises((qmlp.QmlpError, RuntimeError, ValueError, TypeError), match=match):
            call()


@gpu
def test_function_transforms_and_tangents_are_refused():
    x, offsets = torch.randn(2, 3, 40, device="cuda"), torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    weight = tokens.quantise_mx4(torch.randn(2, 5, 40, device="cuda"))
    rows = tokens.quantise_mx4(x)
    for call in (lambda v: tokens.quantise_mx4(v).codes, lambda v: tokens.mx4_linear(v, weight, offsets)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(torch.autograd.forward_ad.make_dual(x[0], torch.ones_like(x[0])))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda c, s: tokens.Mx4(c, s, 40).dequantise())(rows.codes, rows.scales)
    assert tokens.mx4_linear(x[0], weight, offsets).shape == (3, 5)


def test_tensors_on_the_host_are_refused():
    weight = tokens.Mx4(torch.zeros(1, 5, 16, dtype=torch.uint8), torch.zeros(1, 5, 1, dtype=torch.uint8), 30)
    for call in (lambda: tokens.quantise_mx4(torch.zeros(3, 4)), lambda: weight.dequantise(), lambda: tokens.mx4_linear(torch.zeros(3, 30), weight)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_c_interface_refuses_before_any_launch():
    """Descriptors that do not fit end in a status and a message; nothing of them is read (these calls need no device)."""
    lib, F, H, I, B = _lib.lib, _lib.QMLP_FLOAT, _lib.QMLP_HALF, _lib.QMLP_INT32, _lib.QMLP_UINT8
    none = _lib.TensorDesc()
    x, codes, scales = descriptor(F, 4, 40), descriptor(B, 4, 32), descriptor(B, 4, 2)
    quantise = lambda x, c, s: lib.qmlp_tokens_mx4_quantise(x, c, s, None)  # noqa: E731
    refused(quantise(x, descriptor(F, 4, 32), scales), "must be of type UINT8")
    refused(quantise(x, descriptor(B, 4, 16), descriptor(B, 4, 1)), "must have 2 entries")
    refused(quantise(x, descriptor(B, 4, 31), scales), "16 bytes for each")
    refused(quantise(descriptor(F, 5, 40), codes, scales), "must have 5 entries")
    refused(quantise(x, descriptor(B, 4, 32, strides=(31, 1)), scales), "share memory")
    refused(quantise(x, codes, descriptor(B, 4, 2, strides=(4, 2))), "consecutive")
    refused(quantise(descriptor(B, 4, 40), codes, scales), "float, half or bfloat16")
    refused(quantise(descriptor(F, 1, 2 ** 31 - 2 ** 12 + 1), codes, scales), "columns must not be more")
    refused(lib.qmlp_tokens_mx4_values(codes, scales, descriptor(F, 4, 65), None), "must have 3 entries")
    refused(lib.qmlp_tokens_mx4_values(codes, descriptor(B, 3, 2), x, None), "of one size")
    w, s, off, y = descriptor(B, 3, 5, 32), descriptor(B, 3, 5, 2), descriptor(I, 4), descriptor(F, 4, 5)
    linear = lambda *a: lib.qmlp_tokens_mx4_linear(*a)  # noqa: E731
    many, ymany = descriptor(F, 400, 40), descriptor(F, 400, 5)
    refused(linear(many, none, w, s, off, none, ymany, None, None), "bytes of memory")
    refused(linear(many, none, w, s, off, none, ymany, 264, None), "aligned")
    refused(linear(x, none, w, s, none, none, y, 256, None), "one expert")
    refused(linear(descriptor(F, 4, 65), none, w, s, off, none, y, 256, None), "2 blocks")
    refused(linear(codes, scales, descriptor(B, 3, 5, 48), descriptor(B, 3, 5, 3), off, none, y, 256, None), "3 blocks")
    refused(linear(x, none, w, s, off, none, descriptor(H, 4, 5), 256, None), "must be of type FLOAT")
    refused(linear(x, none, w, s, off, descriptor(H, 3, 5), y, 256, None), "must be of type FLOAT")
    refused(linear(x, none, w, s, off, none, descriptor(F, 4, 5, strides=(4, 1)), 256, None), "share memory")
    refused(linear(x, none, descriptor(B, 3, 0, 32), descriptor(B, 3, 0, 2), off, none, descriptor(F, 4, 0), 256, None), "inputs and outputs")
    refused(linear(descriptor(F, 2 ** 31 - 1, 40, strides=(0, 1)), none, w, s, off, none, descriptor(F, 2 ** 31 - 1, 5), 256, None), "rows must not be more")
    refused(lib.qmlp_tokens_mx4_linear_memory(-1, 4, 4, 4, ctypes.byref(ctypes.c_size_t())), "must not be negative")


def test_other_entry_points_refuse_bytes():
    out = ctypes.c_void_p()
    assert _lib.lib.qmlp_activation_create(b"relu", ctypes.byref(out)) == 0
    d = descriptor(_lib.QMLP_UINT8, 4, 6)
    refused(_lib.lib.qmlp_activation_forward(out, d, d, None), "unknown tensor precision")
    _lib.check(_lib.lib.qmlp_activation_destroy(out))
    refused(_lib.lib.qmlp_tokens_layer_norm(d, _lib.TensorDesc(), _lib.TensorDesc(), 1e-5, d, _lib.TensorDesc(), _lib.TensorDesc(), None), "float, half or bfloat16")
