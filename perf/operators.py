"""A mixture of experts and its optimizer, operator by operator: the router (top-k of softmax or sigmoid scores, with a
balancing bias and groups), the gated feed-forward products of the chosen experts, and the orthogonalised momentum
update of weight matrices, each with its gradient where a program trains through it.

A case is a dict of plain values; `prepare` makes what a program holds before the call, as torch tensors on the GPU;
`run` makes one pass. Where `own` is false the pass is computed by elementary torch operations, otherwise by this
framework, which takes the tensors where they are. Expert numbers are floats, as indices are throughout the framework's
API; they are compared as whole numbers. `exact` is the same pass in 64 bits from the definitions.
"""

import math

import numpy as np
import torch

own = False


class Results(dict):
    """Results by name. A framework tensor is handed to torch, without a copy, when its entry is read; expert numbers
    become integers then."""

    def __getitem__(self, name):
        value = dict.__getitem__(self, name)
        if not isinstance(value, torch.Tensor):
            value = torch.from_dlpack(value.detach())
        return value.long() if name == "chosen" else value


def listed():
    return [
        # The router of one new token of a served model: sigmoid scores, a balancing bias, half of the groups kept.
        {"name": "route_token", "kind": "route", "tokens": 1, "experts": 64, "top_k": 4, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "renormalise": True, "train": False},
        # A training batch of a plain router: softmax, the two best, weights that sum to one.
        {"name": "route_batch", "kind": "route", "tokens": 4096, "experts": 64, "top_k": 2, "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renormalise": True, "train": True},
        # Sizes that fit no vector or wavefront; the weights are the softmax's own.
        {"name": "route_odd", "kind": "route", "tokens": 999, "experts": 33, "top_k": 5, "score": "softmax", "bias": True,
         "groups": 1, "top_groups": 1, "renormalise": False, "train": True},
        # The router over a long batch of many small experts.
        {"name": "route_long", "kind": "route", "tokens": 65536, "experts": 256, "top_k": 8, "score": "sigmoid",
         "bias": True, "groups": 8, "top_groups": 4, "renormalise": True, "train": True},
        # One new token through its two experts: bound by reading their weights.
        {"name": "experts_token", "kind": "experts", "tokens": 1, "experts": 16, "top_k": 2, "width": 1024,
         "hidden": 4096, "train": False},
        # A few tokens served together, many small experts: a row or two for each.
        {"name": "experts_decode", "kind": "experts", "tokens": 16, "experts": 64, "top_k": 6, "width": 1024,
         "hidden": 512, "train": False},
        # A train step whose sizes fit no tile and no 16-byte row.
        {"name": "experts_odd", "kind": "experts", "tokens": 999, "experts": 5, "top_k": 2, "width": 131, "hidden": 515,
         "train": True},
        # A train step over a long batch with few large experts.
        {"name": "experts_step", "kind": "experts", "tokens": 8192, "experts": 8, "top_k": 2, "width": 1024,
         "hidden": 4096, "train": True},
        # A train step over a long batch with many small experts.
        {"name": "experts_fine", "kind": "experts", "tokens": 8192, "experts": 64, "top_k": 6, "width": 1024,
         "hidden": 512, "train": True},
        # The update of a digit classifier's matrices: launches and latency.
        {"name": "muon_digits", "kind": "muon", "shapes": "784x256,256x10", "steps": 5, "raw": False},
        # The update of the benchmark's three weight matrices.
        {"name": "muon_mlp", "kind": "muon", "shapes": "1024x4096,4096x4096,4096x1000", "steps": 5, "raw": False},
        # Every expert's matrix of a layer orthogonalised by itself.
        {"name": "orthogonal_experts", "kind": "muon", "shapes": "16x1024x512", "steps": 5, "raw": True},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


_MOST_ROUTED = 65536 * 256
_MOST_PRODUCT = 16384 * 1024 * 4096
_MOST_WEIGHTS = 64 * 1024 * 512
_MOST_MUON = 4096 ** 3


def draw(rng):
    kind = rng.choice(["route", "experts", "muon"])
    if kind == "route":
        while True:
            tokens, experts = _log_int(rng, 1, 65536), _log_int(rng, 4, 256)
            if tokens * experts <= _MOST_ROUTED:
                break
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if experts % g == 0])
        top_groups = rng.randint(1, groups)
        return {"kind": kind, "tokens": tokens, "experts": experts,
                "top_k": rng.randint(1, min(8, experts // groups * top_groups)), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "renormalise": rng.random() < 0.7, "train": rng.random() < 0.7}
    if kind == "experts":
        while True:
            train = rng.random() < 0.6
            tokens, experts = _log_int(rng, 1, 8192 if train else 512), _log_int(rng, 2, 64)
            top_k, width, hidden = rng.randint(1, min(6, experts)), _log_int(rng, 32, 2048), _log_int(rng, 32, 4096)
            if tokens * top_k * width * hidden <= _MOST_PRODUCT and experts * width * hidden <= _MOST_WEIGHTS:
                return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": top_k, "width": width,
                        "hidden": hidden, "train": train}
    while True:
        shapes = [[_log_int(rng, 2, 4096), _log_int(rng, 2, 4096)] for _ in range(rng.choice([1, 1, 2, 3]))]
        if rng.random() < 0.4:
            shapes = [[_log_int(rng, 2, 32)] + s for s in shapes[:1]]
        if sum(math.prod(s) * min(s[-2:]) for s in shapes) <= _MOST_MUON and sum(map(math.prod, shapes)) <= 4096 * 6000:
            return {"kind": kind, "shapes": ",".join("x".join(map(str, s)) for s in shapes), "steps": 5,
                    "raw": rng.random() < 0.4}


def _shapes(case):
    return [[int(n) for n in s.split("x")] for s in case["shapes"].split(",")]


LEARNING_RATE, MOMENTUM, WEIGHT_DECAY = 0.02, 0.95, 0.01
# The quintic of the iteration: x -> a x + b x^3 + c x^5 on every singular value.
QUINTIC = (3.4445, -4.7750, 2.0315)


# ---- inputs ------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale

    state = {"case": dict(case)}
    if case["kind"] == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        # Logits of a router that has begun to specialise: some experts are liked more than others.
        state["logits"] = normal(tokens, experts) + normal(experts, scale=0.5)
        state["bias"] = normal(experts, scale=0.02) if case["bias"] else None
        state["dweights"] = normal(tokens, top_k, scale=1e-3) if case["train"] else None
    elif case["kind"] == "experts":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        width, hidden = case["width"], case["hidden"]
        logits = normal(tokens, experts) + normal(experts, scale=0.5)
        best = torch.topk(logits, top_k, dim=1)
        state["chosen"] = best.indices.float()
        state["weights"] = torch.softmax(best.values, 1)
        state["x"] = normal(tokens, width)
        for name, rows, cols in (("gate", width, hidden), ("up", width, hidden), ("down", hidden, width)):
            state[name] = (torch.rand(experts, rows, cols, generator=gen, device="cuda") * 2 - 1) * (3.0 / rows) ** 0.5
        state["dy"] = normal(tokens, width, scale=1.0 / tokens) if case["train"] else None
    else:
        for i, shape in enumerate(_shapes(case)):
            state["g%d" % i] = normal(*shape, scale=1e-3)
            if not case["raw"]:
                state["p%d" % i] = (torch.rand(*shape, generator=gen, device="cuda") * 2 - 1) * shape[-2] ** -0.5
                state["m%d" % i] = normal(*shape, scale=3e-3)
    return state


# ---- one pass in the framework --------------------------------------------------


def _own_route(state):
    import vectorcore_amd as vc
    case = state["case"]
    given = [t for t in (state["logits"], state["bias"], state["dweights"]) if t is not None]
    given = list(vc.from_dlpack(*given))
    logits = given.pop(0)
    bias = given.pop(0) if case["bias"] else None
    logits.requires_grad = case["train"]
    weights, chosen = vc.route(logits, case["top_k"], bias=bias, score=case["score"], groups=case["groups"],
                               top_groups=case["top_groups"], renormalise=case["renormalise"])
    result = Results(weights=weights, chosen=chosen)
    if case["train"]:
        weights.backward(given.pop(0))
        result["dlogits"] = logits.grad
    return result


def _own_experts(state):
    import vectorcore_amd as vc
    case = state["case"]
    names = ["x", "weights", "gate", "up", "down", "chosen"] + (["dy"] if case["train"] else [])
    v = dict(zip(names, vc.from_dlpack(*(state[n] for n in names))))
    leaves = names[:5] if case["train"] else []
    for name in leaves:
        v[name].requires_grad = True
    plan = vc.ExpertPlan(v["chosen"], case["experts"])
    hidden = vc.expert_gated(v["x"], v["gate"], v["up"], plan)
    rows = vc.expert_linear(hidden, v["down"], plan, ordered=True)
    y = vc.expert_combine(rows, v["weights"], plan)
    result = Results(y=y)
    if case["train"]:
        y.backward(v["dy"])
        result.update(("d" + name, v[name].grad) for name in leaves)
    return result


def _own_muon(state):
    import vectorcore_amd as vc
    case = state["case"]
    count = len(_shapes(case))
    if case["raw"]:
        given = vc.from_dlpack(*(state["g%d" % i] for i in range(count)))
        return Results(("o%d" % i, vc.orthogonalise(g, steps=case["steps"])) for i, g in enumerate(given))
    given = vc.from_dlpack(*(state[n + str(i)] for n in "pmg" for i in range(count)))
    params, momenta, grads = given[:count], given[count:2 * count], given[2 * count:]
    vc.muon_step(params, momenta, LEARNING_RATE, momentum=MOMENTUM, weight_decay=WEIGHT_DECAY, steps=case["steps"],
                 grads=grads)
    result = Results(("p%d" % i, p) for i, p in enumerate(params))
    result.update(("m%d" % i, m) for i, m in enumerate(momenta))
    return result


# ---- one pass in elementary torch operations ----------------------------------------


def _scores(logits, score):
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_route(state):
    case, logits = state["case"], state["logits"]
    tokens, experts = logits.shape
    # The choice is made next to borders between scores: in 64 bits.
    ranked = _scores(logits.double(), case["score"])
    if state["bias"] is not None:
        ranked = ranked + state["bias"].double()
    if case["groups"] > 1:
        grouped = ranked.view(tokens, case["groups"], -1)
        best = torch.topk(grouped, min(2, grouped.shape[2]), dim=2).values.sum(2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        ranked = torch.where(open_[:, :, None], grouped, -math.inf).view(tokens, experts)
    chosen = torch.sort(ranked, dim=1, descending=True, stable=True).indices[:, :case["top_k"]].contiguous()
    scores = _scores(logits, case["score"])
    picked = torch.gather(scores, 1, chosen)
    total = picked.sum(1, keepdim=True)
    weights = picked / total if case["renormalise"] else picked
    result = {"weights": weights, "chosen": chosen}
    if case["train"]:
        d = state["dweights"]
        if case["renormalise"]:
            d = (d - (d * weights).sum(1, keepdim=True)) / total
        if case["score"] == "sigmoid":
            dlogits = torch.zeros_like(scores).scatter_(1, chosen, d * picked * (1 - picked))
        else:
            dscores = torch.zeros_like(scores).scatter_(1, chosen, d)
            dlogits = scores * (dscores - (d * picked).sum(1, keepdim=True))
        result["dlogits"] = dlogits
    return result


def _plain_experts(state):
    """The rows of each expert side by side, as a batch of matrices padded to the longest."""
    case, x, weights = state["case"], state["x"], state["weights"]
    train = case["train"]
    (tokens, top_k), experts, width = weights.shape, case["experts"], case["width"]
    flat = state["chosen"].long().flatten()
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=experts)
    longest = int(counts.max())
    expert = flat[order]
    slot = expert * longest + torch.arange(len(order), device=x.device) - (torch.cumsum(counts, 0) - counts)[expert]
    token = order // top_k
    rows = x.new_zeros(experts * longest, width)
    rows[slot] = x[token]
    rows = rows.view(experts, longest, width)
    gate, up, down = state["gate"], state["up"], state["down"]
    g, u = rows @ gate, rows @ up
    s = 1 / (1 + torch.exp(-g))
    h = g * s * u
    z = (h @ down).view(-1, width)
    place = torch.empty_like(slot)
    place[order] = slot
    mine = z[place].view(tokens, top_k, width)
    y = (weights[:, :, None] * mine).sum(1)
    result = {"y": y}
    if train:
        dy = state["dy"]
        result["dweights"] = (dy[:, None, :] * mine).sum(2)
        dz = x.new_zeros(experts * longest, width)
        dz[place] = (weights[:, :, None] * dy[:, None, :]).view(-1, width)
        dz = dz.view(experts, longest, width)
        dh = dz @ down.transpose(1, 2).contiguous()
        result["ddown"] = h.transpose(1, 2).contiguous() @ dz
        du = dh * g * s
        dg = dh * u * (s + g * s * (1 - s))
        across = rows.transpose(1, 2).contiguous()
        result["dgate"], result["dup"] = across @ dg, across @ du
        dx = (dg @ gate.transpose(1, 2).contiguous() + du @ up.transpose(1, 2).contiguous()).view(-1, width)
        result["dx"] = dx[place].view(tokens, top_k, width).sum(1)
    return result


def _orthogonal(g, steps):
    x = g if g.shape[-2] <= g.shape[-1] else g.transpose(-2, -1).contiguous()
    norm = x.square().sum((-2, -1), keepdim=True).sqrt()
    x = x / norm.clamp(min=torch.finfo(torch.float32).tiny)
    a, b, c = QUINTIC
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x if g.shape[-2] <= g.shape[-1] else x.transpose(-2, -1).contiguous()


def _plain_muon(state):
    case, result = state["case"], {}
    for i, shape in enumerate(_shapes(case)):
        g = state["g%d" % i]
        if case["raw"]:
            result["o%d" % i] = _orthogonal(g, case["steps"])
            continue
        p, m = state["p%d" % i], state["m%d" % i]
        m.mul_(MOMENTUM).add_(g)
        update = _orthogonal(g + MOMENTUM * m, case["steps"])
        rate = LEARNING_RATE * max(1.0, shape[-1] / shape[-2]) ** 0.5
        p.mul_(1 - LEARNING_RATE * WEIGHT_DECAY).sub_(rate * update)
        result["p%d" % i], result["m%d" % i] = p, m
    return result


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"route": _own_route, "experts": _own_experts, "muon": _own_muon}[kind](state)
    return {"route": _plain_route, "experts": _plain_experts, "muon": _plain_muon}[kind](state)


# ---- what a pass cannot do without ---------------------------------------------


def work(case):
    if case["kind"] == "route":
        elements, picks = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        extra = case["experts"] * case["bias"]
        if case["train"]:
            return {"bytes": 4 * (2 * elements + 3 * picks + extra), "flops": 10 * elements}
        return {"bytes": 4 * (elements + 2 * picks + extra), "flops": 6 * elements}
    if case["kind"] == "experts":
        tokens, width, hidden = case["tokens"], case["width"], case["hidden"]
        picks = tokens * case["top_k"]
        matrix = 3 * width * hidden
        # Every weight that a token reads; every weight's gradient is written.
        reached = min(case["experts"], picks) * matrix
        if case["train"]:
            return {"bytes": 4 * (4 * tokens * width + 3 * picks + reached + case["experts"] * matrix),
                    "flops": 6 * picks * matrix}
        return {"bytes": 4 * (2 * tokens * width + 2 * picks + reached), "flops": 2 * picks * matrix}
    elements = flops = 0
    for shape in _shapes(case):
        short, long = sorted(shape[-2:])
        matrices = math.prod(shape[:-2])
        elements += math.prod(shape)
        # The gram matrix and its square are symmetric: half of each is computed.
        flops += matrices * case["steps"] * (3 * short * short * long + short ** 3)
    return {"bytes": 4 * elements * (2 if case["raw"] else 5), "flops": flops}


# ---- the same pass in 64 bits, from the definitions --------------------------------


def _exact_route(case, state):
    logits = state["logits"].cpu().numpy().astype(np.float64)
    tokens, experts = logits.shape
    if case["score"] == "sigmoid":
        scores = 1 / (1 + np.exp(-logits))
    else:
        scores = np.exp(logits - logits.max(1, keepdims=True))
        scores /= scores.sum(1, keepdims=True)
    ranked = scores if state["bias"] is None else scores + state["bias"].cpu().numpy().astype(np.float64)
    rows = np.arange(tokens)
    if case["groups"] > 1:
        grouped = np.sort(ranked.reshape(tokens, case["groups"], -1), axis=2)
        strength = grouped[:, :, -2:].sum(2)
        ranked = ranked.copy().reshape(tokens, case["groups"], -1)
        closed = np.ones((tokens, case["groups"]), dtype=bool)
        for _ in range(case["top_groups"]):
            best = strength.argmax(1)
            strength[rows, best] = -np.inf
            closed[rows, best] = False
        ranked[closed] = -np.inf
        ranked = ranked.reshape(tokens, experts)
    left = ranked.copy()
    chosen = np.empty((tokens, case["top_k"]), dtype=np.int64)
    for j in range(case["top_k"]):
        chosen[:, j] = left.argmax(1)  # the first of equals
        left[rows, chosen[:, j]] = -np.inf
    picked = np.take_along_axis(scores, chosen, 1)
    total = picked.sum(1, keepdims=True) if case["renormalise"] else np.ones((tokens, 1))
    result = {"weights": picked / total, "chosen": chosen}
    if case["train"]:
        d = state["dweights"].cpu().numpy().astype(np.float64)
        dpicked = d / total
        if case["renormalise"]:
            dpicked = dpicked - (d * picked).sum(1, keepdims=True) / total ** 2
        dscores = np.zeros_like(scores)
        np.put_along_axis(dscores, chosen, dpicked, 1)
        if case["score"] == "sigmoid":
            result["dlogits"] = dscores * scores * (1 - scores)
        else:
            result["dlogits"] = scores * (dscores - (dscores * scores).sum(1, keepdims=True))
    return result


def _exact_experts(case, state):
    v = {k: t.double() for k, t in state.items() if isinstance(t, torch.Tensor)}
    leaves = ("x", "weights", "gate", "up", "down")
    for name in leaves:
        v[name].requires_grad_(case["train"])
    y = torch.zeros_like(v["x"])
    for e in range(case["experts"]):  # every expert computes its own tokens and adds them up
        token, j = torch.nonzero(state["chosen"] == e, as_tuple=True)
        rows = v["x"][token]
        hidden = torch.nn.functional.silu(rows @ v["gate"][e]) * (rows @ v["up"][e])
        y = y.index_add(0, token, v["weights"][token, j][:, None] * (hidden @ v["down"][e]))
    result = {"y": y.detach()}
    if case["train"]:
        grads = torch.autograd.grad(y, [v[name] for name in leaves], v["dy"])
        result.update(("d" + name, g) for name, g in zip(leaves, grads))
    return result


def _exact_muon(case, state):
    result = {}
    a, b, c = QUINTIC
    for i, shape in enumerate(_shapes(case)):
        g = state["g%d" % i].double()
        u = g
        if not case["raw"]:
            m = MOMENTUM * state["m%d" % i].double() + g
            u = g + MOMENTUM * m
        o = u / torch.linalg.matrix_norm(u, keepdim=True)
        wide = shape[-2] <= shape[-1]
        for _ in range(case["steps"]):
            if wide:
                gram = o @ o.mT
                o = a * o + b * (gram @ o) + c * (gram @ (gram @ o))
            else:
                gram = o.mT @ o
                o = a * o + b * (o @ gram) + c * ((o @ gram) @ gram)
        if case["raw"]:
            result["o%d" % i] = o
            continue
        p = state["p%d" % i].double() * (1 - LEARNING_RATE * WEIGHT_DECAY)
        result["p%d" % i] = p - LEARNING_RATE * math.sqrt(max(1.0, shape[-1] / shape[-2])) * o
        result["m%d" % i] = m
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "experts": _exact_experts, "muon": _exact_muon}[case["kind"]](case, state)
