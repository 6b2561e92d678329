"""Operators around the experts of a token model: the work that a user of ``qmlp.tokens`` has them do beside ``perf/operators.py``.

Families and where their sizes come from:

* ``route``     the router's choice: softmax over the experts, the largest few of it with their experts, and the gradient of the
                logits: a decoded batch, a training step of a layer with many experts
* ``dispatch``  every token's row to the places of its experts, and the gradient of the rows (widths as in ``perf/operators.py``)
* ``combine``   the rows of a token's experts back at the token, weighted and added up, on top of the token itself; gradients of
                rows, weights and residual
* ``quantise``  numbers of 4 bits in blocks of 32 with a common power of two (MXFP4), and the values they stand for: the weights
                of a layer, rows of odd widths
* ``linear``    the linear layer of every expert with weights of 4 bits, on rows that are quantised in the call: the layers of
                ``perf/operators.py`` as they are served

A case is a dict of plain values; ``op`` is ``forward`` (no gradients) or ``train`` (the forward pass and all gradients, for a
given gradient of the output).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32   # numbers with a common scale


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the tokens of one decoded batch: latency
        {"name": "route_decode", "family": "route", "op": "forward", "rows": 24, "experts": 64, "chosen": 2, "dtype": "bfloat16",
         "normalised": True, "masked": False},
        # a training step of a layer with many experts
        {"name": "route_train", "family": "route", "op": "train", "rows": 65536, "experts": 128, "chosen": 8, "dtype": "float32",
         "normalised": False, "masked": True},
        # one decoded batch to its experts
        {"name": "dispatch_decode", "family": "dispatch", "op": "forward", "rows": 24, "chosen": 2, "channels": 1024,
         "dtype": "bfloat16", "dropped": 0.0},
        # a training step of a wide model
        {"name": "dispatch_wide_train", "family": "dispatch", "op": "train", "rows": 32768, "chosen": 2, "channels": 2048,
         "dtype": "bfloat16", "dropped": 0.0},
        # the decoded batch back from its experts
        {"name": "combine_decode", "family": "combine", "op": "forward", "rows": 24, "chosen": 2, "channels": 1024,
         "dtype": "bfloat16", "weights": "bfloat16", "residual": True, "dropped": 0.0},
        # an odd width in single precision, tokens that have lost experts
        {"name": "combine_ragged_train", "family": "combine", "op": "train", "rows": 5003, "chosen": 3, "channels": 333,
         "dtype": "float32", "weights": "float32", "residual": False, "dropped": 0.02},
        # a training step of a wide model
        {"name": "combine_wide_train", "family": "combine", "op": "train", "rows": 32768, "chosen": 2, "channels": 2048,
         "dtype": "bfloat16", "weights": "float32", "residual": True, "dropped": 0.0},
        # rows of an odd width in single precision
        {"name": "quantise_ragged", "family": "quantise", "op": "forward", "rows": 4099, "channels": 777, "dtype": "float32"},
        # the weights of a layer of wide experts
        {"name": "quantise_weights", "family": "quantise", "op": "forward", "rows": 16 * 4096, "channels": 2048, "dtype": "bfloat16"},
        # a decoded batch: few rows for each expert, bound by the weights that are read
        {"name": "linear_decode", "family": "linear", "op": "forward", "rows": 24, "experts": 64, "inputs": 1024, "outputs": 4096,
         "dtype": "bfloat16", "bias": False, "skew": 1.0, "ungrouped": 0},
        # odd widths in single precision, some rows without an expert
        {"name": "linear_ragged", "family": "linear", "op": "forward", "rows": 5003, "experts": 12, "inputs": 333, "outputs": 200,
         "dtype": "float32", "bias": True, "skew": 1.0, "ungrouped": 37},
        # the first layer of the experts of a wide model on long prompts
        {"name": "linear_wide", "family": "linear", "op": "forward", "rows": 32768, "experts": 16, "inputs": 2048, "outputs": 4096,
         "dtype": "bfloat16", "bias": False, "skew": 0.5, "ungrouped": 0},
    ]


def _log_uniform(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n))


def _width(rng, low, high):
    """Half of the widths are multiples of 16, as models have them, half are any number."""
    n = _log_uniform(rng, low, high)
    return max(16, n // 16 * 16) if rng.random() < 0.5 and high >= 16 else n


def draw(rng):
    family = rng.choice(["route", "dispatch", "combine", "combine", "quantise", "linear", "linear", "linear"])
    op = "forward" if family in ("quantise", "linear") else rng.choice(["forward", "train"])
    case = {"family": family, "op": op}
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if family == "route":
        experts = _log_uniform(rng, 2, 512)
        case.update(rows=_log_uniform(rng, 1, min(65536, (1 << 23) // experts)), experts=experts,
                    chosen=rng.randint(1, min(8, experts)), dtype=dtype, normalised=rng.random() < 0.5, masked=rng.random() < 0.5)
    elif family in ("dispatch", "combine"):
        channels, chosen = _width(rng, 16, 4096), rng.randint(1, 8)
        rows = _log_uniform(rng, 1, min(65536, (1 << 27) // (channels * chosen)))
        case.update(rows=rows, chosen=chosen, channels=channels, dtype=dtype, dropped=rng.choice([0.0, 0.0, 0.02]))
        if family == "combine":
            case.update(weights=rng.choice(["float32", dtype]), residual=rng.random() < 0.5)
    elif family == "quantise":
        channels = _width(rng, 16, 8192)
        case.update(rows=_log_uniform(rng, 1, min(65536, (1 << 27) // channels)), channels=channels, dtype=dtype)
    else:
        inputs, outputs = _width(rng, 16, 4096), _width(rng, 16, 4096)
        # the plain form pads every expert's rows to the longest: less than the largest listed case in any event
        most = 2.0 * 32768 * 2048 * 4096 / 8
        rows = _log_uniform(rng, 1, int(min(65536, max(2, most / (2.0 * inputs * outputs)))))
        experts = _log_uniform(rng, 1, max(1, min(256, (1 << 27) // (inputs * outputs))))
        case.update(rows=rows, experts=experts, inputs=inputs, outputs=outputs, dtype=dtype, bias=rng.random() < 0.5,
                    skew=rng.choice([0.0, 0.5, 1.0]), ungrouped=rng.choice([0, 0, rows // 50]))
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _places(g, rows, chosen, dropped):
    """Where the rows of every token lie among those of all experts: every token has different experts, of random preference;
    -1 - place where the token has lost an expert, whose rows come last."""
    experts = max(16, 2 * chosen)
    score = _normal(g, rows, experts) + _normal(g, experts)
    index = torch.argsort(score, 1, descending=True)[:, :chosen]
    index = torch.where(torch.rand(rows, chosen, device="cuda", generator=g) < dropped, experts, index).flatten()
    order = torch.sort(index, stable=True)[1]
    places = torch.empty_like(order)
    places[order] = torch.arange(len(order), device=order.device)
    return torch.where(index < experts, places, -1 - places).view(rows, chosen).int()


def prepare(case, seed):
    g = _generator(seed)
    family, rows, train = case["family"], case["rows"], case["op"] == "train"
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if family == "route":
        logits = 1.5 * _normal(g, rows, case["experts"]) + 0.5 * _normal(g, case["experts"])
        if case["masked"]:   # experts that a row must not take, padded rows that take none
            logits[torch.rand(rows, case["experts"], device="cuda", generator=g) < 0.05] = -math.inf
            logits[torch.rand(rows, device="cuda", generator=g) < 0.01] = -math.inf
        state["logits"] = logits.to(dtype)
        if train:
            state["grad"] = _normal(g, rows, case["chosen"]).to(dtype)
    elif family in ("dispatch", "combine"):
        chosen, channels = case["chosen"], case["channels"]
        state["places"] = _places(g, rows, chosen, case["dropped"])
        if family == "dispatch":
            state["x"] = _normal(g, rows, channels).to(dtype)
            if train:
                state["grad"] = _normal(g, rows * chosen, channels).to(dtype)
        else:
            state["rows"] = _normal(g, rows * chosen, channels).to(dtype)
            state["weights"] = torch.softmax(_normal(g, rows, chosen), 1).to(DTYPES[case["weights"]])
            if case["residual"]:
                state["residual"] = _normal(g, rows, channels).to(dtype)
            if train:
                state["grad"] = _normal(g, rows, channels).to(dtype)
    elif family == "quantise":
        # channels with spreads of their own
        state["x"] = (_normal(g, rows, case["channels"]) * torch.exp(_normal(g, case["channels"]))).to(dtype)
    else:
        experts, inputs, outputs = case["experts"], case["inputs"], case["outputs"]
        # an expert's share of the rows: even, or by random preferences
        preferences = torch.softmax(case["skew"] * _normal(g, experts), 0)
        grouped = max(0, rows - case["ungrouped"])
        chosen = torch.multinomial(preferences, grouped, replacement=True, generator=g) if grouped else preferences.new_zeros(0).long()
        counts = torch.bincount(chosen, minlength=experts)
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        state["longest"] = int(counts.max())   # for programs that pad every expert's rows to the longest
        state["x"] = _normal(g, rows, inputs).to(dtype)
        state["codes"], state["scales"] = _quantised(_normal(g, experts, outputs, inputs) / math.sqrt(inputs))
        if case["bias"]:
            state["bias"] = (0.1 * _normal(g, experts, outputs)).to(dtype)
    if train:
        for name in ("logits", "x", "rows", "weights", "residual"):
            if name in state:
                state[name].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    family, train = state["case"]["family"], state["case"]["op"] == "train"
    if own:
        return _own[family](state, train)
    with torch.no_grad():   # the plain forms have their gradients' formulas
        return _plain[family](state, train)


def _framework():
    # the working folder is the root of the tree that is measured
    path = os.path.abspath("quick-mlp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qmlp
    return qmlp.tokens


def _own_route(s, train):
    weights, index = _framework().route(s["logits"], s["case"]["chosen"], s["case"]["normalised"])
    if not train:
        return {"weights": weights, "index": index}
    logits, = torch.autograd.grad(weights, (s["logits"],), s["grad"])
    return {"weights": weights.detach(), "index": index, "logits": logits}


def _own_dispatch(s, train):
    rows = _framework().dispatch(s["x"], s["places"])
    if not train:
        return {"rows": rows}
    x, = torch.autograd.grad(rows, (s["x"],), s["grad"])
    return {"rows": rows.detach(), "x": x}


def _own_combine(s, train):
    y = _framework().combine(s["rows"], s["places"], s["weights"], s.get("residual"))
    if not train:
        return {"y": y}
    names = ["rows", "weights"] + (["residual"] if "residual" in s else [])
    grads = torch.autograd.grad(y, [s[n] for n in names], s["grad"])
    return {"y": y.detach(), **dict(zip(names, grads))}


def _own_quantise(s, train):
    return {"values": _framework().quantise_mx4(s["x"]).dequantise(s["x"].dtype)}


def _own_linear(s, train):
    tokens = _framework()
    weight = tokens.Mx4(s["codes"], s["scales"], s["case"]["inputs"])
    return {"y": tokens.mx4_linear(s["x"], weight, s["offsets"], s.get("bias"))}


_own = {"route": _own_route, "dispatch": _own_dispatch, "combine": _own_combine, "quantise": _own_quantise, "linear": _own_linear}


def _plain_route(s, train):
    logits, chosen, dtype = s["logits"].float(), s["case"]["chosen"], s["logits"].dtype
    top = logits.max(1, keepdim=True)[0]
    any_ = top > -math.inf
    e = torch.where(any_, torch.exp(logits - torch.where(any_, top, 0.0)), 0.0)
    sorted_, order = torch.sort(logits, dim=1, descending=True, stable=True)
    taken = sorted_[:, :chosen] > -math.inf
    order = order[:, :chosen]
    parts = torch.where(taken, torch.gather(e, 1, order), 0.0)
    total = (parts if s["case"]["normalised"] else e).sum(1, keepdim=True)
    total = torch.where(any_, total, 1.0)
    weights = parts / total
    out = {"weights": weights.to(dtype), "index": torch.where(taken, order, -1).int()}
    if train:
        grad = torch.where(taken, s["grad"].float(), 0.0)
        mean = (grad * weights).sum(1, keepdim=True)
        if s["case"]["normalised"]:
            dense = torch.zeros_like(logits).scatter_(1, order, weights * (grad - mean))
        else:
            dense = e / total * (torch.zeros_like(logits).scatter_(1, order, grad) - mean)
        out["logits"] = dense.to(dtype)
    return out


def _taken(places):
    """Places of the rows and whether the token has them."""
    places = places.long()
    return torch.where(places >= 0, places, -1 - places), places >= 0


def _plain_dispatch(s, train):
    place, taken = _taken(s["places"])
    tokens, chosen = place.shape
    x = s["x"].float()
    rows = torch.zeros((tokens * chosen, x.shape[1]), device=x.device)
    for j in range(chosen):
        rows[place[:, j]] = torch.where(taken[:, j, None], x, 0.0)
    out = {"rows": rows.to(s["x"].dtype)}
    if train:
        grad = s["grad"].float()
        dx = torch.zeros_like(x)
        for j in range(chosen):
            dx += torch.where(taken[:, j, None], grad[place[:, j]], 0.0)
        out["x"] = dx.to(s["x"].dtype)
    return out


def _plain_combine(s, train):
    place, taken = _taken(s["places"])
    rows, weights, dtype = s["rows"].float(), s["weights"].float(), s["rows"].dtype
    y = s["residual"].float() if "residual" in s else torch.zeros((place.shape[0], rows.shape[1]), device=rows.device)
    for j in range(place.shape[1]):
        y = y + torch.where(taken[:, j, None], weights[:, j, None] * rows[place[:, j]], 0.0)
    out = {"y": y.to(dtype)}
    if train:
        grad = s["grad"].float()
        drows, dweights = torch.zeros_like(rows), torch.zeros_like(weights)
        for j in range(place.shape[1]):
            drows[place[:, j]] = torch.where(taken[:, j, None], weights[:, j, None] * grad, 0.0)
            dweights[:, j] = torch.where(taken[:, j], (rows[place[:, j]] * grad).sum(1), 0.0)
        out.update(rows=drows.to(dtype), weights=dweights.to(s["weights"].dtype))
        if "residual" in s:
            out["residual"] = grad.to(dtype)
    return out


def _quantised(x):
    """(..., 16 * blocks) bytes of two codes each, the first in the low bits, and (..., blocks) biased exponents of the scales."""
    blocks = (x.shape[-1] + BLOCK - 1) // BLOCK
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - x.shape[-1])).unflatten(-1, (blocks, BLOCK))
    largest = x.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(largest)[1] - 3   # the largest number, 6, has the exponent 2; frexp's mantissas are below 1
    exponent = torch.where(largest > 0, exponent, -127).clamp(-127, 127)
    v = x.abs().double() * torch.exp2(-exponent.double())   # (in 64 bits: 2^127 times a small number)
    # to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, halfway to the even code
    code = ((v > 0.25).byte() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5)).byte()
    code = (code + 8 * torch.signbit(x).byte()).flatten(-2)
    finite = largest.isfinite()
    return code[..., 0::2] + 16 * code[..., 1::2], torch.where(finite, exponent + 127, 255).byte().squeeze(-1)


def _values(codes, scales, columns):
    """In 32 bits what codes and scales stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2).unflatten(-1, (-1, BLOCK))
    scale = torch.where(scales < 255, torch.exp2(scales.double() - 127), math.nan)
    return (v * scale[..., None]).float().flatten(-2)[..., :columns]


def _plain_quantise(s, train):
    return {"values": _values(*_quantised(s["x"]), s["x"].shape[1]).to(s["x"].dtype)}


def _plain_linear(s, train):
    """Every expert's rows padded to the longest, one batched product over the experts."""
    inputs = s["case"]["inputs"]
    x, weight = _values(*_quantised(s["x"]), inputs), _values(s["codes"], s["scales"], inputs)
    offsets, experts, longest, rows = s["offsets"].long(), weight.shape[0], s["longest"], x.shape[0]
    row = torch.arange(rows, device=x.device)
    expert = torch.searchsorted(offsets, row, right=True) - 1
    # (rows without an expert: to a place behind those of all experts, which is cut off)
    place = torch.where(row < offsets[-1], expert * longest + row - offsets[expert], experts * longest)
    padded = torch.zeros((experts * longest + 1, inputs), device=x.device)
    padded[place] = x
    y = torch.bmm(padded[:-1].view(experts, longest, inputs), weight.transpose(1, 2))
    if "bias" in s:
        y = y + s["bias"].float()[:, None, :]
    y = torch.cat([y.reshape(-1, y.shape[2]), y.new_zeros((1, y.shape[2]))])
    return {"y": y[place].to(s["x"].dtype)}


_plain = {"route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "quantise": _plain_quantise,
          "linear": _plain_linear}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    family, rows, train = case["family"], case["rows"], case["op"] == "train"
    size = DTYPES[case["dtype"]].itemsize
    if family == "route":
        n, chosen = rows * case["experts"], rows * case["chosen"]
        return {"bytes": size * (n + chosen) + 4 * chosen + (size * (n + chosen) if train else 0),
                "flops": n * (4 + case["chosen"]) + (6 * n if train else 0)}
    if family in ("dispatch", "combine"):
        chosen, tokens = rows * case["chosen"], rows * case["channels"]
        moved = chosen * case["channels"]
        if family == "dispatch":
            return {"bytes": (2 if train else 1) * size * (tokens + moved) + 4 * chosen, "flops": max(1, moved if train else 0)}
        weights = DTYPES[case["weights"]].itemsize * chosen
        numbers = moved + tokens * (2 if case["residual"] else 1)
        if train:
            numbers += moved + tokens   # (the residual's gradient is that of the output)
        return {"bytes": size * numbers + weights * (2 if train else 1) + 4 * chosen, "flops": (5 if train else 2) * moved}
    if family == "quantise":
        n = rows * case["channels"]
        return {"bytes": 2 * size * n, "flops": 4 * n}
    inputs, outputs, grouped = case["inputs"], case["outputs"], max(0, rows - case["ungrouped"])
    # experts without rows need no weights
    experts = min(case["experts"], grouped)
    blocks = (inputs + BLOCK - 1) // BLOCK
    numbers = rows * (inputs + outputs) + (experts * outputs if case["bias"] else 0)
    return {"bytes": size * numbers + experts * outputs * blocks * 17 + 4 * (case["experts"] + 1),
            "flops": max(1, 2 * grouped * inputs * outputs)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _exact_values(x):
    """Every block in units of its largest number's power of two: steps of a half below 2, of 1 below 4, of 2 up to 6."""
    columns = x.shape[-1]
    spare = -columns % BLOCK
    v = torch.cat([x, x.new_zeros((*x.shape[:-1], spare))], -1).reshape(*x.shape[:-1], -1, BLOCK)
    largest = v.abs().max(-1, keepdim=True)[0]
    unit = torch.exp2(torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0))))
    unit = torch.where(unit > largest, unit / 2, unit)      # (should the logarithm have been rounded up to a whole number)
    unit = torch.where(unit * 2 <= largest, unit * 2, unit)
    unit = torch.where(largest > 0, unit, 1.0).clamp_min(2.0 ** -125) / 4
    magnitude = v.abs() / unit
    step = torch.where(magnitude < 2, 0.5, torch.where(magnitude < 4, 1.0, 2.0))
    rounded = (torch.round(magnitude / step) * step).clamp_max(6.0)
    return (torch.sign(v) * rounded * unit).reshape(*x.shape[:-1], -1)[..., :columns]


def exact(case, seed):
    s = prepare(case, seed)
    train = case["op"] == "train"
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["family"] == "route":
        logits = d["logits"]
        # the chosen ones one after the other: the largest that is left, the first of equals
        left, index = logits.clone(), []
        for _ in range(case["chosen"]):
            largest = left.max(1, keepdim=True)[0]
            first = torch.where(left == largest, torch.arange(left.shape[1], device=left.device), left.shape[1]).min(1)[0]
            index.append(torch.where(largest[:, 0] > -math.inf, first, -1))
            left.scatter_(1, first[:, None], -math.inf)
        index = torch.stack(index, 1)
        held = torch.zeros(logits.shape[0], logits.shape[1] + 1, dtype=torch.bool, device=logits.device)
        held = held.scatter_(1, torch.where(index >= 0, index, logits.shape[1]), True)[:, :-1]
        over = logits.masked_fill(~held, -math.inf) if case["normalised"] else logits
        p = torch.softmax(over, 1).nan_to_num(0.0)   # (rows without experts)
        gathered = torch.gather(p, 1, index.clamp_min(0)) * (index >= 0)
        out = {"weights": gathered, "index": None}
        if train:
            full = torch.zeros_like(p)
            for j in range(case["chosen"]):
                full.scatter_add_(1, index[:, j:j + 1].clamp_min(0), (d["grad"][:, j] * (index[:, j] >= 0))[:, None])
            out["logits"] = p * full - p * (p * full).sum(1, keepdim=True)
        return out
    if case["family"] in ("dispatch", "combine"):
        flat = s["places"].long().flatten()
        token = torch.arange(case["rows"], device=flat.device).repeat_interleave(case["chosen"])
        has = torch.nonzero(flat >= 0).flatten()
        place, token = flat[has], token[has]
        if case["family"] == "dispatch":
            rows = torch.zeros((case["rows"] * case["chosen"], case["channels"]), dtype=torch.float64, device=flat.device)
            rows[place] = d["x"][token]
            out = {"rows": rows}
            if train:
                out["x"] = torch.zeros_like(d["x"]).index_add_(0, token, d["grad"][place])
            return out
        w = d["weights"].flatten()[has]
        y = d["residual"].clone() if "residual" in d else torch.zeros((case["rows"], case["channels"]), dtype=torch.float64, device=flat.device)
        out = {"y": y.index_add_(0, token, d["rows"][place] * w[:, None])}
        if train:
            drows = torch.zeros_like(d["rows"])
            drows[place] = d["grad"][token] * w[:, None]
            dweights = torch.zeros_like(d["weights"].flatten())
            dweights[has] = (d["grad"][token] * d["rows"][place]).sum(1)
            out.update(rows=drows, weights=dweights.view_as(d["weights"]))
            if "residual" in d:
                out["residual"] = d["grad"]
        return out
    if case["family"] == "quantise":
        return {"values": _exact_values(d["x"])}
    x = _exact_values(d["x"])
    # (the weights are what their codes stand for: sign, exponent and mantissa of two bits, one and one)
    codes = torch.stack([s["codes"] % 16, s["codes"] // 16], -1).flatten(-2).int()
    exponent, mantissa = (codes % 8) // 2, codes % 2
    weight = torch.where(exponent > 0, (2 + mantissa) * torch.exp2(exponent.double() - 2), mantissa * 0.5)
    weight = weight * (1 - 2 * (codes // 8)) * torch.exp2(s["scales"].double() - 127).repeat_interleave(BLOCK, -1)
    weight = weight[..., :case["inputs"]]
    offsets = s["offsets"].tolist()
    y = x.new_zeros((case["rows"], case["outputs"]))
    for e in range(case["experts"]):
        part = slice(offsets[e], offsets[e + 1])
        if offsets[e] < offsets[e + 1]:
            y[part] = x[part] @ weight[e].T
            if "bias" in d:
                y[part] += d["bias"][e]
    return {"y": y}
