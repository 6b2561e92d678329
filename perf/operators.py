"""Operators of a token model with experts: the work that a user of ``qmlp.tokens`` has them do.

Families and where their sizes come from:

* ``group``      rows sorted by the expert (the network, the object) that they belong to: a decoded batch, the samples of an
                 image among the small networks of a scene
* ``embedding``  rows of a learned table by token, times a scale, and the gradient of the table: latent codes per object of
                 the width of this framework's networks (64), a vocabulary in front of a wide model
* ``norm``       layer norm over the channels of every row, and the gradients of input, weight and bias
* ``experts``    the linear layer of every expert on its own rows, and the gradients of input, weights and biases: many
                 64 x 64 layers (the width of this framework's networks), few wide ones

A case is a dict of plain values; ``op`` is ``forward`` (no gradients) or ``train`` (the forward pass and all gradients, for a
given gradient of the output).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
          "int32": torch.int32, "int64": torch.int64}
EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the tokens of one decoded batch among the experts of a layer: launches and the host's path
        {"name": "group_decode", "family": "group", "op": "forward", "rows": 64, "groups": 8, "index": "int64"},
        # the samples of an image among the small networks that a scene is cut into
        {"name": "group_scene", "family": "group", "op": "forward", "rows": 1 << 20, "groups": 4096, "index": "int32"},
        # one token for each of a batch of sequences
        {"name": "embedding_decode", "family": "embedding", "op": "forward", "rows": 32, "vocabulary": 32768,
         "channels": 1024, "dtype": "float16", "index": "int64"},
        # learned codes of a thousand objects or images, trained beside a coordinate network
        {"name": "embedding_codes_train", "family": "embedding", "op": "train", "rows": 20011, "vocabulary": 1000,
         "channels": 64, "dtype": "float32", "index": "int32"},
        # a vocabulary trained on long sequences: few tokens are frequent, most are rare
        {"name": "embedding_vocabulary_train", "family": "embedding", "op": "train", "rows": 65536, "vocabulary": 65536,
         "channels": 1024, "dtype": "bfloat16", "index": "int64"},
        # one decoded token: latency
        {"name": "norm_decode", "family": "norm", "op": "forward", "rows": 1, "channels": 1024, "dtype": "float16"},
        # an odd width in single precision
        {"name": "norm_ragged_train", "family": "norm", "op": "train", "rows": 4099, "channels": 777, "dtype": "float32"},
        # a training step of a wide model
        {"name": "norm_wide_train", "family": "norm", "op": "train", "rows": 32768, "channels": 4096,
         "dtype": "bfloat16"},
        # a layer of many small networks, each trained on the samples of its part of a scene
        {"name": "experts_scene_train", "family": "experts", "op": "train", "rows": 1 << 17, "experts": 512,
         "inputs": 64, "outputs": 64, "dtype": "float16", "bias": True, "skew": 0.5, "ungrouped": 0},
        # a decoded batch: few rows for each expert, bound by the weights that are read
        {"name": "experts_decode", "family": "experts", "op": "forward", "rows": 24, "experts": 64, "inputs": 1024,
         "outputs": 4096, "dtype": "bfloat16", "bias": False, "skew": 1.0, "ungrouped": 0},
        # odd widths in single precision, some rows without an expert
        {"name": "experts_ragged_train", "family": "experts", "op": "train", "rows": 5003, "experts": 12, "inputs": 333,
         "outputs": 200, "dtype": "float32", "bias": True, "skew": 1.0, "ungrouped": 37},
        # the first layer of the experts of a wide model, trained
        {"name": "experts_wide_train", "family": "experts", "op": "train", "rows": 32768, "experts": 16, "inputs": 2048,
         "outputs": 4096, "dtype": "bfloat16", "bias": False, "skew": 0.5, "ungrouped": 0},
    ]


def _log_uniform(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n))


def _width(rng, low, high):
    """Half of the widths are multiples of 16, as models have them, half are any number."""
    n = _log_uniform(rng, low, high)
    return max(16, n // 16 * 16) if rng.random() < 0.5 and high >= 16 else n


def draw(rng):
    family = rng.choice(["group", "embedding", "norm", "norm", "experts", "experts", "experts"])
    op = "forward" if family == "group" else rng.choice(["forward", "train"])
    case = {"family": family, "op": op}
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if family == "group":
        case.update(rows=_log_uniform(rng, 1, 1 << 20), groups=_log_uniform(rng, 1, 4096),
                    index=rng.choice(["int32", "int64"]))
    elif family == "embedding":
        case.update(rows=_log_uniform(rng, 1, 65536), vocabulary=_log_uniform(rng, 16, 65536),
                    channels=_width(rng, 4, 1024), dtype=dtype, index=rng.choice(["int32", "int64"]))
    elif family == "norm":
        channels = _width(rng, 8, 8192)
        case.update(rows=_log_uniform(rng, 1, min(32768, (1 << 27) // channels)), channels=channels, dtype=dtype)
    else:
        inputs, outputs = _width(rng, 16, 2048), _width(rng, 16, 4096)
        # single precision has a smaller part of the work: the largest models are trained in 16 bits
        most = 2.0 * 32768 * 2048 * 4096 / (16 if dtype == "float32" else 2)
        rows = _log_uniform(rng, 1, int(min(1 << 17, max(2, most / (2.0 * inputs * outputs)))))
        experts = _log_uniform(rng, 1, max(1, min(512, (1 << 27) // (inputs * outputs))))
        case.update(rows=rows, experts=experts, inputs=inputs, outputs=outputs, dtype=dtype, bias=rng.random() < 0.5,
                    skew=rng.choice([0.0, 0.5, 1.0]), ungrouped=rng.choice([0, 0, rows // 50]))
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _tokens(g, rows, count, dtype):
    """Token ids with frequencies that fall off as the rank grows, scattered over the vocabulary, 2 % of them padding (-1)."""
    u = torch.rand(rows, device="cuda", generator=g)
    rank = (torch.exp(u * math.log(count + 1)) - 1).long().clamp_(0, count - 1)
    shuffled = torch.randperm(count, device="cuda", generator=g)
    index = shuffled[rank]
    index[torch.rand(rows, device="cuda", generator=g) < 0.02] = -1
    return index.to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    family, rows, train = case["family"], case["rows"], case["op"] == "train"
    state = {"case": case}
    if family == "group":
        # the nearer to one corner of the scene, the more samples a network gets
        u = torch.rand(rows, device="cuda", generator=g)
        index = (u * u * case["groups"]).long().clamp_(0, case["groups"] - 1).to(DTYPES[case["index"]])
        index[torch.rand(rows, device="cuda", generator=g) < 0.01] = -1   # samples outside of the scene
        state["index"] = index
    elif family == "embedding":
        dtype = DTYPES[case["dtype"]]
        state["index"] = _tokens(g, rows, case["vocabulary"], DTYPES[case["index"]])
        state["table"] = (0.02 * _normal(g, case["vocabulary"], case["channels"])).to(dtype)
        state["scale"] = math.sqrt(case["channels"])
        if train:
            state["grad"] = _normal(g, rows, case["channels"]).to(dtype)
    elif family == "norm":
        dtype, channels = DTYPES[case["dtype"]], case["channels"]
        # channels with means and spreads of their own, as the residual stream of a model has them
        x = _normal(g, rows, channels) * (0.5 + 2 * torch.rand(channels, device="cuda", generator=g)) + _normal(g, channels)
        state["x"] = x.to(dtype)
        state["weight"] = (1 + 0.1 * _normal(g, channels)).to(dtype)
        state["bias"] = (0.1 * _normal(g, channels)).to(dtype)
        if train:
            state["grad"] = _normal(g, rows, channels).to(dtype)
    else:
        dtype, experts, inputs, outputs = DTYPES[case["dtype"]], case["experts"], case["inputs"], case["outputs"]
        # an expert's share of the rows: even, or by random preferences
        preferences = torch.softmax(case["skew"] * _normal(g, experts), 0)
        grouped = max(0, rows - case["ungrouped"])
        chosen = torch.multinomial(preferences, grouped, replacement=True, generator=g) if grouped else preferences.new_zeros(0).long()
        counts = torch.bincount(chosen, minlength=experts)
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        state["longest"] = int(counts.max())   # for programs that pad every expert's rows to the longest
        state["x"] = _normal(g, rows, inputs).to(dtype)
        state["weight"] = (_normal(g, experts, outputs, inputs) / math.sqrt(inputs)).to(dtype)
        if case["bias"]:
            state["bias"] = (0.1 * _normal(g, experts, outputs)).to(dtype)
        if train:
            state["grad"] = _normal(g, rows, outputs).to(dtype)
    if train:
        for name in ("table", "x", "weight", "bias"):
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


def _own_group(s, train):
    order, offsets = _framework().group(s["index"], s["case"]["groups"])
    return {"order": order, "offsets": offsets}


def _own_embedding(s, train):
    y = _framework().embedding(s["index"], s["table"], s["scale"])
    if not train:
        return {"y": y}
    table, = torch.autograd.grad(y, (s["table"],), s["grad"])
    return {"y": y.detach(), "table": table}


def _own_norm(s, train):
    y = _framework().layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if not train:
        return {"y": y}
    x, weight, bias = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    return {"y": y.detach(), "x": x, "weight": weight, "bias": bias}


def _own_experts(s, train):
    y = _framework().grouped_linear(s["x"], s["weight"], s["offsets"], s.get("bias"))
    if not train:
        return {"y": y}
    names = ["x", "weight"] + (["bias"] if "bias" in s else [])
    grads = torch.autograd.grad(y, [s[n] for n in names], s["grad"])
    return {"y": y.detach(), **dict(zip(names, grads))}


_own = {"group": _own_group, "embedding": _own_embedding, "norm": _own_norm, "experts": _own_experts}


def _plain_group(s, train):
    groups = s["case"]["groups"]
    index = s["index"].long()
    key = torch.where((index >= 0) & (index < groups), index, groups)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(groups + 1, device=key.device))
    return {"order": order.int(), "offsets": offsets.int()}


def _plain_embedding(s, train):
    index, table, scale = s["index"].long(), s["table"], s["scale"]
    valid = (index >= 0) & (index < table.shape[0])
    index = torch.where(valid, index, 0)
    factor = (scale * valid.float())[:, None]
    out = {"y": (table[index].float() * factor).to(table.dtype)}
    if train:
        grad = torch.zeros(table.shape, device=table.device)
        grad.index_add_(0, index, s["grad"].float() * factor)
        out["table"] = grad.to(table.dtype)
    return out


def _plain_norm(s, train):
    x, weight, bias = s["x"].float(), s["weight"].float(), s["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    normal = centred * rstd
    dtype = s["x"].dtype
    out = {"y": (normal * weight + bias).to(dtype)}
    if train:
        grad = s["grad"].float()
        inner = grad * weight
        dx = rstd * (inner - inner.mean(1, keepdim=True) - normal * (inner * normal).mean(1, keepdim=True))
        out.update(x=dx.to(dtype), weight=(grad * normal).sum(0).to(dtype), bias=grad.sum(0).to(dtype))
    return out


def _plain_experts(s, train):
    """Every expert's rows padded to the longest, one batched product over the experts."""
    x, weight, offsets, dtype = s["x"], s["weight"].float(), s["offsets"].long(), s["x"].dtype
    experts, outputs, inputs = weight.shape
    rows, longest = x.shape[0], s["longest"]
    row = torch.arange(rows, device=x.device)
    expert = torch.searchsorted(offsets, row, right=True) - 1
    # (rows without an expert: to a place behind those of all experts, which is cut off)
    place = torch.where(row < offsets[-1], expert * longest + row - offsets[expert], experts * longest)

    def padded(t):
        p = torch.zeros((experts * longest + 1, t.shape[1]), device=t.device)
        p[place] = t.float()
        p[-1] = 0
        return p[:-1].view(experts, longest, t.shape[1])

    def unpadded(p):
        p = torch.cat([p.reshape(-1, p.shape[2]), p.new_zeros((1, p.shape[2]))])
        return p[place]

    xp = padded(x)
    y = torch.bmm(xp, weight.transpose(1, 2))
    if "bias" in s:
        y = y + s["bias"].float()[:, None, :]
    out = {"y": unpadded(y).to(dtype)}
    if train:
        gp = padded(s["grad"])
        out["x"] = unpadded(torch.bmm(gp, weight)).to(dtype)
        out["weight"] = torch.bmm(gp.transpose(1, 2), xp).to(dtype)
        if "bias" in s:
            out["bias"] = gp.sum(1).to(dtype)
    return out


_plain = {"group": _plain_group, "embedding": _plain_embedding, "norm": _plain_norm, "experts": _plain_experts}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    family, rows, train = case["family"], case["rows"], case["op"] == "train"
    if family == "group":
        return {"bytes": rows * (4 + DTYPES[case["index"]].itemsize) + 4 * (case["groups"] + 1), "flops": rows}
    size = DTYPES[case["dtype"]].itemsize
    if family == "embedding":
        channels, vocabulary = case["channels"], case["vocabulary"]
        # distinct tokens among the rows: their frequencies fall off as 1 / (rank + 1)
        norm = math.log(vocabulary + 1)
        distinct = sum(1 - (1 - math.log1p(1 / (r + 1)) / norm) ** rows for r in range(vocabulary))
        bytes_ = rows * DTYPES[case["index"]].itemsize + size * channels * (distinct + rows)
        if train:
            bytes_ += size * channels * (rows + vocabulary)
        return {"bytes": int(bytes_), "flops": rows * channels * (2 if train else 1)}
    if family == "norm":
        n, channels = rows * case["channels"], case["channels"]
        # forward: x -> y; training: dy besides, dx
        return {"bytes": size * ((4 if train else 2) * n + (4 if train else 2) * channels), "flops": (19 if train else 7) * n}
    inputs, outputs, grouped = case["inputs"], case["outputs"], max(0, rows - case["ungrouped"])
    # experts without rows need no weights in the forward pass
    preferences = min(case["experts"], grouped)
    weights, biases = inputs * outputs, outputs if case["bias"] else 0
    numbers = rows * (inputs + outputs) + preferences * (weights + biases)
    flops = 2 * grouped * weights
    if train:
        numbers += rows * (inputs + outputs) + case["experts"] * (weights + biases)
        flops *= 3
    return {"bytes": size * numbers + 4 * (case["experts"] + 1), "flops": max(1, flops)}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["family"] == "group":
        return None   # whole numbers
    s = prepare(case, seed)
    train = case["op"] == "train"
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["family"] == "embedding":
        index = s["index"].long()
        y = torch.zeros((index.numel(), case["channels"]), dtype=torch.float64, device=index.device)
        used = torch.nonzero((index >= 0) & (index < case["vocabulary"])).flatten()
        y[used] = d["table"][index[used]] * s["scale"]
        out = {"y": y}
        if train:
            # sums of consecutive rows in the order of the tokens, as differences of running sums
            tokens, order = torch.sort(index[used])
            running = (d["grad"][used][order] * s["scale"]).cumsum(0)
            running = torch.cat([running.new_zeros((1, running.shape[1])), running])
            ends = torch.searchsorted(tokens, torch.arange(case["vocabulary"] + 1, device=tokens.device))
            out["table"] = running[ends[1:]] - running[ends[:-1]]
        return out
    if case["family"] == "norm":
        x, weight, bias = d["x"], d["weight"], d["bias"]
        n = x.shape[1]
        mean = x.sum(1) / n
        variance = (x * x).sum(1) / n - mean * mean
        sigma = torch.sqrt(variance + EPS)
        normal = (x - mean[:, None]) / sigma[:, None]
        out = {"y": normal * weight + bias}
        if train:
            grad = d["grad"]
            h = grad * weight
            correction = (h.sum(1)[:, None] + normal * (h * normal).sum(1)[:, None]) / n
            out.update(x=(h - correction) / sigma[:, None], weight=torch.einsum("rc,rc->c", grad, normal), bias=grad.sum(0))
        return out
    offsets = s["offsets"].tolist()
    y = d["x"].new_zeros((case["rows"], case["outputs"]))
    out = {"y": y}
    if train:
        out["x"] = torch.zeros_like(d["x"])
        out["weight"] = torch.zeros_like(d["weight"])
        if "bias" in d:
            out["bias"] = torch.zeros_like(d["bias"])
    for e in range(case["experts"]):
        part = slice(offsets[e], offsets[e + 1])
        if offsets[e] == offsets[e + 1]:
            continue
        y[part] = d["x"][part] @ d["weight"][e].T
        if "bias" in d:
            y[part] += d["bias"][e]
        if train:
            out["x"][part] = d["grad"][part] @ d["weight"][e]
            out["weight"][e] = d["grad"][part].T @ d["x"][part]
            if "bias" in d:
                out["bias"][e] = d["grad"][part].sum(0)
    return out
