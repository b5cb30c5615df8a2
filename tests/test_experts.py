"""The expert products of a mixture of experts against float64: the plan that sorts the picks, both products, the sum of
a token's picks, all gradients, empty experts, dropped picks, odd sizes, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


def layout(chosen, experts):
    """(row of each pick, expert of each row, token of each row), dropped picks last with expert `experts`."""
    flat = chosen.reshape(-1)
    whole = (flat >= 0) & (flat < experts) & (flat == np.trunc(flat))
    group = np.where(whole, np.nan_to_num(flat), experts).astype(int)
    order = np.argsort(group, kind="stable")
    place = np.empty_like(order)
    place[order] = np.arange(len(order))
    return place, group[order], order // chosen.shape[1]


def picks(rng, tokens, top_k, experts, kind):
    c = rng.integers(0, experts, (tokens, top_k)).astype(np.float32)
    if kind == "one":
        c[:] = experts // 2
    elif kind == "skewed":
        c = np.minimum(c, rng.integers(0, experts, (tokens, top_k))).astype(np.float32)
    elif kind == "dropped" and c.size:
        flat = c.reshape(-1)
        bad = np.array([-1, experts, np.nan, 0.5, np.inf, -np.inf, 1e30, 2 ** 32], np.float32)
        at = rng.random(flat.size) < 0.4
        flat[at] = bad[rng.integers(0, len(bad), at.sum())]
    elif kind == "all dropped":
        c[:] = -1
    return c


def bound(*factors):
    """A sum of k products, each factor's own error counted: (k + 8) roundings of the products of magnitudes."""
    return UNIT * sum(k + 8 for k in factors)


def gated_unit(x, gate, up, down, weights, chosen, dy):
    """y and every gradient in float64, and for each a bound of a float32 chain's error: the same chain on magnitudes, in
    which silu is at most its argument, its slope at most 1.1 and its curvature at most 0.5."""
    experts, width, hidden = gate.shape
    x, gate, up, down, weights, dy = (a.astype(np.float64) for a in (x, gate, up, down, weights, dy))
    place, group, token = layout(chosen, experts)
    tokens, top_k = chosen.shape
    rows = len(group)
    out = {n: np.zeros_like(a) for n, a in dict(y=x, x=x, gate=gate, up=up, down=down, weights=weights).items()}
    mag = {n: np.zeros_like(a) for n, a in out.items()}
    flat_w, pick = weights.reshape(-1), np.empty(rows, int)
    pick[place] = np.arange(rows)
    most = max((np.bincount(group, minlength=experts + 1)[:experts]).max() if rows else 0, 1)
    for e in range(experts):
        r = np.nonzero(group == e)[0]
        if not len(r):
            continue
        t, p = token[r], pick[r]
        xe, w, d = x[t], flat_w[p][:, None], dy[t]
        g, u = xe @ gate[e], xe @ up[e]
        s = 1 / (1 + np.exp(-g))
        h = g * s * u
        z = h @ down[e]
        dz = w * d
        dh = dz @ down[e].T
        du, dg = dh * g * s, dh * u * (s + g * s * (1 - s))
        np.add.at(out["y"], t, w * z)
        out["weights"].reshape(-1)[p] = (d * z).sum(1)
        out["down"][e], out["gate"][e], out["up"][e] = h.T @ dz, xe.T @ dg, xe.T @ du
        np.add.at(out["x"], t, dg @ gate[e].T + du @ up[e].T)
        a = np.abs
        mg, mu = a(xe) @ a(gate[e]), a(xe) @ a(up[e])
        mh = mg * mu
        mz, mdz = mh @ a(down[e]), a(dz)
        mdh = mdz @ a(down[e]).T
        mdu, mdg = mdh * mg, mdh * mu * (1.1 + 0.5 * mg)
        np.add.at(mag["y"], t, a(w) * mz)
        mag["weights"].reshape(-1)[p] = (a(d) * mz).sum(1)
        mag["down"][e], mag["gate"][e], mag["up"][e] = mh.T @ mdz, a(xe).T @ mdg, a(xe).T @ mdu
        np.add.at(mag["x"], t, mdg @ a(gate[e]).T + mdu @ a(up[e]).T)
    forward = bound(width, width, width, hidden) + 24 * UNIT
    back = bound(width, width, width, hidden, width, hidden, most, top_k, hidden) + 64 * UNIT
    for n in mag:
        mag[n] = mag[n] * (forward + bound(top_k) if n == "y" else back) + 1e-37
    return out, mag


SIZES = [(1, 2, 1, 1, 1), (1, 16, 2, 32, 64), (16, 64, 6, 36, 20), (5, 3, 2, 7, 9), (33, 5, 2, 67, 131), (64, 8, 2, 64, 64),
         (129, 4, 1, 128, 65), (200, 7, 3, 100, 96), (300, 3, 2, 160, 260), (77, 1, 1, 33, 31), (700, 2, 2, 48, 40),
         (40, 130, 4, 20, 24), (0, 4, 2, 8, 8), (6, 4, 2, 300, 5), (9, 4, 2, 5, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["even", "one", "skewed", "dropped", "all dropped"])
@pytest.mark.parametrize("tokens,experts,top_k,width,hidden", SIZES)
def test_gated_unit(tokens, experts, top_k, width, hidden, kind, device):
    rng = np.random.default_rng(tokens + 7 * experts + width + len(kind))
    f = lambda *s, scale=1.0: (scale * rng.standard_normal(s)).astype(np.float32)
    v = dict(x=f(tokens, width), gate=f(experts, width, hidden, scale=width ** -0.5),
             up=f(experts, width, hidden, scale=width ** -0.5), down=f(experts, hidden, width, scale=hidden ** -0.5),
             weights=np.abs(f(tokens, top_k)))
    dy, chosen = f(tokens, width), picks(rng, tokens, top_k, experts, kind)
    t = {n: vc.Tensor(a, requires_grad=True, device=device) for n, a in v.items()}
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), experts)
    assert (plan.tokens, plan.top_k, plan.experts, plan.rows) == (tokens, top_k, experts, tokens * top_k)
    h = vc.expert_gated(t["x"], t["gate"], t["up"], plan)
    rows = vc.expert_linear(h, t["down"], plan, ordered=True)
    y = vc.expert_combine(rows, t["weights"], plan)
    y.backward(vc.Tensor(dy, device=device))
    want, near = gated_unit(**v, chosen=chosen, dy=dy)
    got = dict({n: a.grad for n, a in t.items()}, y=y)
    for n in want:
        assert tuple(got[n].shape) == want[n].shape
        assert (np.abs(got[n].numpy().reshape(want[n].shape) - want[n]) <= near[n]).all(), n
    dropped = layout(chosen, experts)[1] == experts
    for part in (h, rows):
        assert (part.numpy()[dropped] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ordered", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k,width,columns", [(9, 3, 2, 17, 21), (150, 4, 2, 64, 128), (3, 40, 3, 40, 44),
                                                               (260, 2, 1, 130, 70), (1, 1, 1, 1, 1)])
def test_linear(tokens, experts, top_k, width, columns, ordered, device):
    rng = np.random.default_rng(tokens + width)
    chosen = picks(rng, tokens, top_k, experts, "dropped" if tokens % 2 else "even")
    place, group, token = layout(chosen, experts)
    x = rng.standard_normal((len(group) if ordered else tokens, width)).astype(np.float32)
    w = rng.standard_normal((experts, width, columns)).astype(np.float32)
    g = rng.standard_normal((len(group), columns)).astype(np.float32)
    tx, tw = vc.Tensor(x, requires_grad=True, device=device), vc.Tensor(w, requires_grad=True, device=device)
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), experts)
    y = vc.expert_linear(tx, tw, plan, ordered=ordered)
    y.backward(vc.Tensor(g, device=device))
    x64, w64, g64 = x.astype(np.float64), w.astype(np.float64), g.astype(np.float64)
    want, mag = np.zeros((len(group), columns)), np.zeros((len(group), columns))
    dx, mdx, dw, mdw = np.zeros_like(x64), np.zeros_like(x64), np.zeros_like(w64), np.zeros_like(w64)
    for r, e in enumerate(group):
        if e == experts:
            continue
        s = r if ordered else token[r]
        want[r], mag[r] = x64[s] @ w64[e], np.abs(x64[s]) @ np.abs(w64[e])
        dx[s] += w64[e] @ g64[r]
        mdx[s] += np.abs(w64[e]) @ np.abs(g64[r])
        dw[e] += np.outer(x64[s], g64[r])
        mdw[e] += np.outer(np.abs(x64[s]), np.abs(g64[r]))
    assert (np.abs(y.numpy() - want) <= bound(width) * mag).all()
    assert (np.abs(tx.grad.numpy() - dx) <= bound(columns, top_k) * mdx).all()
    assert (np.abs(tw.grad.numpy() - dw) <= bound(len(group)) * mdw).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens,experts,top_k,width,hidden,kind", [(90, 2, 1, 1100, 60, "skewed"), (70, 1, 1, 70, 1290, "even"),
                                                                    (44, 3, 3, 600, 700, "dropped"), (3000, 3, 1, 40, 70, "skewed")])
def test_long_sums_of_few_tiles(tokens, experts, top_k, width, hidden, kind, device):
    """Sums that are split over workgroups."""
    test_gated_unit(tokens, experts, top_k, width, hidden, kind, device)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k,width,columns", [(4099, 3, 2, 33, 2050), (4099, 3, 2, 2051, 33),
                                                               (45, 5, 2, 2050, 2053), (9000, 6, 1, 96, 1024)])
def test_many_tiles(tokens, experts, top_k, width, columns):
    """Enough tiles for the whole chip: wide ones, each die its share, experts of unequal sizes, one without rows."""
    rng = np.random.default_rng(tokens + width)
    chosen = picks(rng, tokens, top_k, experts - 1, "skewed")
    place, group, token = layout(chosen, experts)
    x, w = rng.standard_normal((tokens, width)).astype(np.float32), rng.standard_normal((experts, width, columns)).astype(np.float32)
    u, g = rng.standard_normal((experts, width, columns)).astype(np.float32), rng.standard_normal((len(group), columns)).astype(np.float32)
    t = [vc.Tensor(a, requires_grad=True, device="hip") for a in (x, w)]
    plan = vc.ExpertPlan(vc.Tensor(chosen, device="hip"), experts)
    y = vc.expert_linear(*t, plan)
    y.backward(vc.Tensor(g, device="hip"))
    h = vc.expert_gated(t[0].detach(), t[1].detach(), vc.Tensor(u, device="hip"), plan).numpy()
    y, dx, dw = y.numpy(), t[0].grad.numpy(), t[1].grad.numpy()
    want_dx, mag_dx = np.zeros(x.shape), np.zeros(x.shape)
    for e in range(experts):
        r = np.nonzero(group == e)[0]
        xe, ge, we, ue = (a.astype(np.float64) for a in (x[token[r]], g[r], w[e], u[e]))
        a, b, mag, mag_u = xe @ we, xe @ ue, np.abs(xe) @ np.abs(we), np.abs(xe) @ np.abs(ue)
        assert (np.abs(y[r] - a) <= bound(width) * mag).all()
        assert (np.abs(h[r] - a / (1 + np.exp(-a)) * b) <= (bound(width, width, width) + 24 * UNIT) * mag * mag_u).all()
        assert (np.abs(dw[e] - xe.T @ ge) <= bound(len(r)) * (np.abs(xe).T @ np.abs(ge))).all()
        np.add.at(want_dx, token[r], ge @ we.T)
        np.add.at(mag_dx, token[r], np.abs(ge) @ np.abs(we).T)
    assert (np.abs(dx - want_dx) <= bound(columns, top_k) * mag_dx).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    rng = np.random.default_rng(5)
    tokens, experts, top_k, width, hidden = 4, 3, 2, 5, 6
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    v = dict(x=f(tokens, width), gate=f(experts, width, hidden), up=f(experts, width, hidden), down=f(experts, hidden, width),
             weights=f(tokens, top_k))
    dy, chosen = f(tokens, width), picks(rng, tokens, top_k, experts, "even")

    def loss(values):
        a = {n: t.astype(np.float64) for n, t in values.items()}
        total = 0.0
        for i in range(tokens):
            for j in range(top_k):
                e = int(chosen[i, j])
                g = a["x"][i] @ a["gate"][e]
                z = (g / (1 + np.exp(-g)) * (a["x"][i] @ a["up"][e])) @ a["down"][e]
                total += a["weights"][i, j] * (z * dy[i]).sum()
        return total

    t = {n: vc.Tensor(a, requires_grad=True, device=device) for n, a in v.items()}
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), experts)
    y = vc.expert_combine(vc.expert_linear(vc.expert_gated(t["x"], t["gate"], t["up"], plan), t["down"], plan, ordered=True),
                          t["weights"], plan)
    y.backward(vc.Tensor(dy, device=device))
    for n, a in v.items():
        for at in {tuple(rng.integers(0, s) for s in a.shape) for _ in range(6)}:
            values = []
            for sign in (1, -1):
                moved = {k: b.astype(np.float64) for k, b in v.items()}
                moved[n][at] += sign * 1e-5
                values.append(loss(moved))
            assert abs(t[n].grad.numpy()[at] - (values[0] - values[1]) / 2e-5) <= 2e-4, n


@pytest.mark.parametrize("device", DEVICES)
def test_only_the_gradients_asked_for(device):
    rng = np.random.default_rng(6)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)
    chosen = picks(rng, 10, 2, 3, "even")
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), 3)
    values = [f(10, 8), f(3, 8, 12), f(3, 8, 12)]
    want = None
    for mask in range(1, 8):
        t = [vc.Tensor(a, requires_grad=bool(mask >> i & 1), device=device) for i, a in enumerate(values)]
        vc.expert_gated(*t, plan).sum().backward()
        grads = [a.grad.numpy() if a.grad is not None else None for a in t]
        assert [g is not None for g in grads] == [bool(mask >> i & 1) for i in range(3)]
        want = want or {}
        for i, g in enumerate(grads):
            if g is not None:
                np.testing.assert_array_equal(g, want.setdefault(i, g))


@pytest.mark.parametrize("device", DEVICES)
def test_not_a_number_stays_in_its_rows(device):
    rng = np.random.default_rng(8)
    chosen = np.array([[0, 1], [1, 2], [2, 0], [3, -1]], np.float32)
    x = rng.standard_normal((4, 40)).astype(np.float32)
    w = rng.standard_normal((4, 40, 36)).astype(np.float32)
    x[1, 3], x[2, 5], w[3, 0, 0] = np.nan, np.inf, -np.inf
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), 4)
    y = vc.expert_linear(vc.Tensor(x, device=device), vc.Tensor(w, device=device), plan).numpy()
    place, group, token = layout(chosen, 4)
    with np.errstate(all="ignore"):
        for r, e in enumerate(group):
            want = (x[token[r]].astype(np.float64) @ w[e].astype(np.float64)) if e < 4 else np.zeros(36)
            finite = np.isfinite(want)
            assert np.isfinite(y[r][finite]).all()
            np.testing.assert_array_equal(np.isnan(y[r]), np.isnan(want))
            np.testing.assert_array_equal(y[r][np.isinf(want)], want[np.isinf(want)])


@pytest.mark.parametrize("device", DEVICES)
def test_wide_ranges_of_magnitude(device):
    """Every product keeps its own precision: rows, columns and single terms many orders of magnitude apart."""
    rng = np.random.default_rng(9)
    tokens, width, columns = 70, 96, 80
    x = rng.standard_normal((tokens, width)) * 10.0 ** rng.integers(-12, 12, (tokens, width))
    w = rng.standard_normal((1, width, columns)) * 10.0 ** rng.integers(-12, 12, (1, width, columns))
    x[3, 1:], w[0, 0, 5] = 0.0, 0.0
    x, w = x.astype(np.float32), w.astype(np.float32)
    plan = vc.ExpertPlan(vc.Tensor(np.zeros((tokens, 1), np.float32), device=device), 1)
    y = vc.expert_linear(vc.Tensor(x, device=device), vc.Tensor(w, device=device), plan).numpy()
    x64, w64 = x.astype(np.float64), w[0].astype(np.float64)
    assert (np.abs(y - x64 @ w64) <= bound(width) * (np.abs(x64) @ np.abs(w64))).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("picks_count,experts", [(1, 1), (511, 3), (512, 64), (513, 64), (3000, 257), (70000, 1024)])
def test_the_plan_keeps_the_order_of_equal_experts(picks_count, experts, device):
    rng = np.random.default_rng(picks_count)
    chosen = picks(rng, picks_count, 1, experts, "dropped")
    plan = vc.ExpertPlan(vc.Tensor(chosen, device=device), experts)
    # Expert matrices of one element that are one: each row is its token's value.
    x = np.arange(picks_count, dtype=np.float32)[:, None] + 1
    rows = vc.expert_linear(vc.Tensor(x, device=device), vc.Tensor.ones((experts, 1, 1), device=device), plan).numpy()
    place, group, token = layout(chosen, experts)
    np.testing.assert_array_equal(rows[:, 0], np.where(group < experts, token + 1, 0))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z = lambda *s: vc.Tensor.zeros(s, device=device)
    for shape in ((3,), (3, 0), (1, 2, 3)):
        with pytest.raises(ValueError):
            vc.ExpertPlan(z(*shape), 4)
    for experts in (0, 1025):
        with pytest.raises(ValueError):
            vc.ExpertPlan(z(3, 2), experts)
    plan = vc.ExpertPlan(z(3, 2), 4)
    for x, w, ordered in ((z(4, 5), z(4, 5, 6), False), (z(3, 5), z(4, 5, 6), True), (z(3, 5), z(3, 5, 6), False),
                          (z(3, 5), z(4, 6, 6), False), (z(3, 5), z(4, 5), False), (z(3), z(4, 5, 6), False)):
        with pytest.raises(ValueError):
            vc.expert_linear(x, w, plan, ordered=ordered)
        with pytest.raises(ValueError):
            vc.expert_gated(x, w, w, plan, ordered=ordered)
    with pytest.raises(ValueError):
        vc.expert_gated(z(3, 5), z(4, 5, 6), z(4, 5, 7), plan)
    for rows, weights in ((z(5, 7), z(3, 2)), (z(6, 7), z(2, 3)), (z(6, 7), z(6))):
        with pytest.raises(ValueError):
            vc.expert_combine(rows, weights, plan)


@pytest.mark.gpu
def test_refuses_a_plan_of_another_device():
    plan = vc.ExpertPlan(vc.Tensor.zeros((3, 2)), 4)
    with pytest.raises(ValueError, match="is on"):
        vc.expert_linear(vc.Tensor.zeros((3, 5), device="hip"), vc.Tensor.zeros((4, 5, 6), device="hip"), plan)
