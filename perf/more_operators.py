"""The ends of a layer and the end of a model, operator by operator: layer normalisation over the last axis, dropout whose
mask is computed from a counter and never stored, and the softmax cross entropy of a linear layer's logits that are never
kept, each with its gradient where a program trains through it.

A case is a dict of plain values; `prepare` makes what a program holds before the call, as torch tensors on the GPU;
`run` makes one pass. Where `own` is false the pass is computed by elementary torch operations, otherwise by this
framework, which takes the tensors where they are. Class numbers are floats, as indices are throughout the framework's
API, and a number that is no class leaves its row out of the loss. `exact` is the same pass in 64 bits from the definitions.
"""

import math

import numpy as np
import torch

own = False


class Results(dict):
    """Results by name. A framework tensor is handed to torch, without a copy, when its entry is read."""

    def __getitem__(self, name):
        value = dict.__getitem__(self, name)
        return value if isinstance(value, torch.Tensor) else torch.from_dlpack(value.detach())


def listed():
    return [
        # One new token of a served model: latency of a single small row.
        {"name": "norm_token", "kind": "norm", "rows": 1, "width": 4096, "affine": True, "train": False},
        # The residual stream of a training batch.
        {"name": "norm_batch", "kind": "norm", "rows": 8192, "width": 4096, "affine": True, "train": True},
        # Rows that fit no vector and no wavefront.
        {"name": "norm_odd", "kind": "norm", "rows": 999, "width": 515, "affine": True, "train": True},
        # Many short rows: a norm over each head's share of the stream, without a weight.
        {"name": "norm_heads", "kind": "norm", "rows": 262144, "width": 64, "affine": False, "train": True},
        # The branch of a training batch, dropped out as it joins the residual stream.
        {"name": "dropout_join", "kind": "dropout", "rows": 8192, "width": 4096, "p": 0.1, "residual": True, "train": True},
        # The hidden layer of a digit classifier: a small launch each way.
        {"name": "dropout_digits", "kind": "dropout", "rows": 256, "width": 256, "p": 0.5, "residual": False, "train": True},
        # A count of elements that is no multiple of the generator's four.
        {"name": "dropout_odd", "kind": "dropout", "rows": 999, "width": 515, "p": 0.25, "residual": True, "train": True},
        # The loss of a digit classifier's last layer.
        {"name": "loss_digits", "kind": "loss", "rows": 256, "width": 256, "classes": 10, "bias": True, "ignored": 0.0,
         "reduction": "mean", "train": True},
        # The score of one token: bound by reading the weights.
        {"name": "loss_token", "kind": "loss", "rows": 1, "width": 1024, "classes": 50000, "bias": False, "ignored": 0.0,
         "reduction": "none", "train": False},
        # The scores of a batch of answers, token by token; a quarter is padding.
        {"name": "loss_score", "kind": "loss", "rows": 2048, "width": 1024, "classes": 50000, "bias": False,
         "ignored": 0.25, "reduction": "none", "train": False},
        # A train step with a weight for each token, sizes that fit no tile.
        {"name": "loss_odd", "kind": "loss", "rows": 999, "width": 515, "classes": 10007, "bias": True, "ignored": 0.1,
         "reduction": "none", "train": True},
        # A train step over a long batch and a large vocabulary.
        {"name": "loss_step", "kind": "loss", "rows": 8192, "width": 1024, "classes": 50000, "bias": False,
         "ignored": 0.1, "reduction": "mean", "train": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


_MOST_ELEMENTS = 8192 * 4096
_MOST_PRODUCT = 8192 * 1024 * 50000
_MOST_SCORED = 2048 * 1024 * 50000
_MOST_WEIGHTS = 1024 * 50000


def draw(rng):
    kind = rng.choice(["norm", "dropout", "loss"])
    train = rng.random() < 0.7
    if kind == "loss":
        while True:
            rows, width, classes = _log_int(rng, 1, 8192), _log_int(rng, 8, 2048), _log_int(rng, 2, 65536)
            if rows * width * classes <= (_MOST_PRODUCT if train else _MOST_SCORED) and width * classes <= _MOST_WEIGHTS:
                return {"kind": kind, "rows": rows, "width": width, "classes": classes, "bias": rng.random() < 0.5,
                        "ignored": rng.choice([0.0, 0.1, 0.5]), "reduction": rng.choice(["mean", "none"]), "train": train}
    while True:
        rows, width = _log_int(rng, 1, 262144), _log_int(rng, 2, 16384)
        if rows * width <= _MOST_ELEMENTS:
            break
    if kind == "norm":
        return {"kind": kind, "rows": rows, "width": width, "affine": rng.random() < 0.7, "train": train}
    return {"kind": kind, "rows": rows, "width": width, "p": rng.uniform(0.02, 0.9), "residual": rng.random() < 0.5,
            "train": train}


EPSILON = 1e-5


# ---- inputs ------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, width = case["rows"], case["width"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale

    state = {"case": dict(case)}
    if case["kind"] == "norm":
        # A stream with a mean of its own and features of unequal size.
        state["x"] = normal(rows, width) * (1 + normal(width, scale=0.3)) + normal(rows, 1, scale=0.5)
        if case["affine"]:
            state["weight"] = 1 + normal(width, scale=0.1)
            state["bias"] = normal(width, scale=0.1)
    elif case["kind"] == "dropout":
        state["x"] = normal(rows, width)
        state["residual"] = normal(rows, width) if case["residual"] else None
        # The generator's seed, and the number of the call's own stream of it.
        state["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x1234567) % 2 ** 63
        state["stream"] = seed % 1000 + 2 ** 33
    else:
        classes = case["classes"]
        state["weight"] = normal(width, classes, scale=width ** -0.5)
        # Frequent classes have low numbers; the model is surer of some rows than of others.
        targets = (torch.rand(rows, generator=gen, device="cuda").pow(3) * classes).long().clamp(max=classes - 1)
        sure = torch.rand(rows, 1, generator=gen, device="cuda") * 12
        state["x"] = normal(rows, width) + sure * state["weight"][:, targets].t()
        left_out = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
        state["targets"] = torch.where(left_out, -1.0, targets.float())
        state["bias"] = normal(classes, scale=0.5) if case["bias"] else None
    if case["train"]:
        if case["kind"] != "loss":
            state["dy"] = normal(rows, width, scale=1.0 / rows)
        elif case["reduction"] == "none":
            state["dy"] = torch.rand(rows, generator=gen, device="cuda") / rows
    return state


# ---- one pass in the framework --------------------------------------------------


def _given(state, names):
    import vectorcore_amd as vc
    names = [n for n in names if state.get(n) is not None]
    return vc, dict(zip(names, vc.from_dlpack(*(state[n] for n in names))))


def _with_gradients(result, y, v, dy, leaves):
    if dy is None:
        y.backward()
    else:
        y.backward(dy)
    result.update(("d" + name, v[name].grad) for name in leaves)
    return result


def _own_norm(state):
    vc, v = _given(state, ["x", "weight", "bias", "dy"])
    train = state["case"]["train"]
    leaves = [n for n in ("x", "weight", "bias") if n in v] if train else []
    for name in leaves:
        v[name].requires_grad = True
    y = vc.layer_norm(v["x"], v.get("weight"), v.get("bias"), eps=EPSILON)
    result = Results(y=y)
    return _with_gradients(result, y, v, v["dy"], leaves) if train else result


def _own_dropout(state):
    vc, v = _given(state, ["x", "residual", "dy"])
    case = state["case"]
    leaves = [n for n in ("x", "residual") if n in v] if case["train"] else []
    for name in leaves:
        v[name].requires_grad = True
    y = vc.dropout(v["x"], case["p"], state["seed"], stream=state["stream"], residual=v.get("residual"))
    result = Results(y=y)
    return _with_gradients(result, y, v, v["dy"], leaves) if case["train"] else result


def _own_loss(state):
    vc, v = _given(state, ["x", "weight", "targets", "bias", "dy"])
    case = state["case"]
    leaves = [n for n in ("x", "weight", "bias") if n in v] if case["train"] else []
    for name in leaves:
        v[name].requires_grad = True
    loss = vc.linear_cross_entropy(v["x"], v["weight"], v["targets"], bias=v.get("bias"), reduction=case["reduction"])
    result = Results(loss=loss)
    return _with_gradients(result, loss, v, v.get("dy"), leaves) if case["train"] else result


# ---- one pass in elementary torch operations ----------------------------------------


def _plain_norm(state):
    case, x = state["case"], state["x"]
    centred = x - x.mean(1, keepdim=True)
    scale = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPSILON)
    normed = centred * scale
    y = normed * state["weight"] + state["bias"] if case["affine"] else normed
    result = {"y": y}
    if case["train"]:
        dy = state["dy"]
        d = dy * state["weight"] if case["affine"] else dy
        result["dx"] = scale * (d - d.mean(1, keepdim=True) - normed * (d * normed).mean(1, keepdim=True))
        if case["affine"]:
            result["dweight"] = (dy * normed).sum(0)
            result["dbias"] = dy.sum(0)
    return result


_WORD = 2 ** 32 - 1
_FACTORS = (0xD2511F53, 0xCD9E8D57)
_STEPS = (0x9E3779B9, 0xBB67AE85)


def _high(factor, word):
    """The upper 32 bits of the product of two 32-bit numbers that int64 holds."""
    return ((factor >> 16) * word + ((factor & 0xFFFF) * word >> 16)) >> 16


def _kept(count, p, seed, stream, device):
    """Philox 4x32 with ten rounds (Salmon et al., 2011): element i is word i % 4 of counter (i / 4, stream), 64 bits each."""
    counter = torch.arange((count + 3) // 4, device=device)
    a, b = counter & _WORD, counter >> 32
    c = torch.full_like(counter, stream & _WORD)
    d = torch.full_like(counter, stream >> 32)
    k, l = seed & _WORD, seed >> 32
    for _ in range(10):
        a, b, c, d = (_high(_FACTORS[1], c) ^ b ^ k, _FACTORS[1] * c & _WORD, _high(_FACTORS[0], a) ^ d ^ l,
                      _FACTORS[0] * a & _WORD)
        k, l = (k + _STEPS[0]) & _WORD, (l + _STEPS[1]) & _WORD
    words = torch.stack([a, b, c, d], 1).flatten()[:count]
    return words >= round(p * 2 ** 32)


def _plain_dropout(state):
    case, x = state["case"], state["x"]
    kept = _kept(x.numel(), case["p"], state["seed"], state["stream"], x.device).view_as(x)
    scale = 1 / (1 - case["p"])
    y = torch.where(kept, x * scale, 0.0)
    if case["residual"]:
        y = state["residual"] + y
    result = {"y": y}
    if case["train"]:
        result["dx"] = torch.where(kept, state["dy"] * scale, 0.0)
        if case["residual"]:
            result["dresidual"] = state["dy"]
    return result


def _plain_loss(state):
    case, x, weight, targets = state["case"], state["x"], state["weight"], state["targets"].long()
    logits = x @ weight
    if case["bias"]:
        logits = logits + state["bias"]
    counted = targets >= 0
    at = targets.clamp(min=0)[:, None]
    shifted = logits - logits.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    each = torch.where(counted, (torch.log(total) - torch.gather(shifted, 1, at))[:, 0], 0.0)
    number = counted.sum().clamp(min=1)
    result = {"loss": each.sum() / number if case["reduction"] == "mean" else each}
    if case["train"]:
        share = 1.0 / number if case["reduction"] == "mean" else state["dy"]
        share = torch.where(counted, share, 0.0)[:, None]
        d = e / total * share
        d.scatter_add_(1, at, -share)
        result["dx"] = d @ weight.t()
        result["dweight"] = x.t() @ d
        if case["bias"]:
            result["dbias"] = d.sum(0)
    return result


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "dropout": _own_dropout, "loss": _own_loss}[kind](state)
    return {"norm": _plain_norm, "dropout": _plain_dropout, "loss": _plain_loss}[kind](state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    rows, width = case["rows"], case["width"]
    elements = rows * width
    if case["kind"] == "norm":
        # x and y; for a gradient dy and dx too, and x again once the gradient of y is known.
        vectors = 2 * width * case["affine"]
        if case["train"]:
            return {"bytes": 4 * (5 * elements + 2 * vectors), "flops": 18 * elements}
        return {"bytes": 4 * (2 * elements + vectors), "flops": 8 * elements}
    if case["kind"] == "dropout":
        passes = 2 + case["residual"] + (2 + case["residual"]) * case["train"]
        return {"bytes": 4 * passes * elements, "flops": (1 + case["train"]) * elements}
    weights, extra = width * case["classes"], rows + case["classes"] * case["bias"]
    if case["train"]:
        return {"bytes": 4 * (2 * elements + 2 * weights + 2 * extra), "flops": 6 * rows * weights}
    return {"bytes": 4 * (elements + weights + extra + rows), "flops": 2 * rows * weights}


# ---- the same pass in 64 bits, from the definitions --------------------------------


def _exact_norm(case, state):
    v = {n: t.double().requires_grad_(case["train"]) for n, t in state.items() if n in ("x", "weight", "bias")}
    x = v["x"]
    deviation = x - x.sum(1)[:, None] / case["width"]
    variance = deviation.pow(2).sum(1)[:, None] / case["width"]
    y = deviation / (variance + EPSILON).sqrt()
    if case["affine"]:
        y = torch.addcmul(v["bias"], y, v["weight"])
    result = {"y": y.detach()}
    if case["train"]:
        names = [n for n in ("x", "weight", "bias") if n in v]
        grads = torch.autograd.grad(y, [v[n] for n in names], state["dy"].double())
        result.update(("d" + n, g) for n, g in zip(names, grads))
    return result


def _exact_dropout(case, state):
    count, mask = state["x"].numel(), np.uint64(2 ** 32 - 1)
    half = np.uint64(32)
    key = [state["seed"] & 0xFFFFFFFF, state["seed"] >> 32]
    blocks = np.arange(-(-count // 4), dtype=np.uint64)
    word = [blocks & mask, blocks >> half, np.full_like(blocks, state["stream"] & 0xFFFFFFFF),
            np.full_like(blocks, state["stream"] >> 32)]
    for r in range(10):
        first, second = np.uint64(0xD2511F53) * word[0], np.uint64(0xCD9E8D57) * word[2]
        keys = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        word = [(second >> half) ^ word[1] ^ keys[0], second & mask, (first >> half) ^ word[3] ^ keys[1], first & mask]
    drawn = np.stack(word, axis=1).reshape(-1)[:count]
    kept = torch.from_numpy(drawn / 2.0 ** 32 >= round(case["p"] * 2 ** 32) / 2.0 ** 32).cuda().view_as(state["x"])
    factor = kept.double() / (1.0 - case["p"])
    y = state["x"].double() * factor
    if case["residual"]:
        y += state["residual"].double()
    result = {"y": y}
    if case["train"]:
        result["dx"] = state["dy"].double() * factor
        if case["residual"]:
            result["dresidual"] = state["dy"].double()
    return result


def _exact_loss(case, state):
    x, weight = state["x"].double(), state["weight"].double()
    bias = state["bias"].double() if case["bias"] else None
    counted = state["targets"] >= 0
    mean, number = case["reduction"] == "mean", max(1, int(counted.sum()))
    loss = torch.zeros(case["rows"], dtype=torch.float64, device=x.device)
    dx, dweight = torch.zeros_like(x), torch.zeros_like(weight)
    dbias = torch.zeros(case["classes"], dtype=torch.float64, device=x.device)
    for rows in torch.nonzero(counted)[:, 0].split(1024):
        target = state["targets"][rows].long()
        logits = torch.addmm(bias, x[rows], weight) if case["bias"] else x[rows] @ weight
        logp = torch.log_softmax(logits, 1)
        loss[rows] = -logp[torch.arange(len(rows)), target]
        if case["train"]:
            d = logp.exp()
            d[torch.arange(len(rows)), target] -= 1
            d *= 1.0 / number if mean else state["dy"][rows].double()[:, None]
            dx[rows] = d @ weight.t()
            dweight += x[rows].t() @ d
            dbias += d.sum(0)
    result = {"loss": loss.sum() / number if mean else loss}
    if case["train"]:
        result.update(dx=dx, dweight=dweight)
        if case["bias"]:
            result["dbias"] = dbias
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "dropout": _exact_dropout, "loss": _exact_loss}[case["kind"]](case, state)
