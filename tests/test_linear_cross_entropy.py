"""The cross entropy of a linear layer against its definition in float64: losses and gradients of either reduction, rows that
are left out, classes without a chance, sure rows, host targets, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


def exact(x, w, t, b, share):
    """Losses, gradients and, of each, how far float32 arithmetic may be off: a sum of k products walks by roundings of its
    terms, 4 sqrt(k) of them at eight deviations; an exponential is off by its argument's error and roundings, of which the
    argument's own size counts."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    counted = t >= 0
    x = np.where(counted[:, None], x, 0.0)
    at = np.where(counted, t, 0).astype(int)
    rows = np.arange(len(x))
    z = x @ w + (0 if b is None else b.astype(np.float64))
    walk = lambda k: UNIT * (8 + 4 * np.sqrt(k))
    z_off = walk(x.shape[1]) * (np.abs(x) @ np.abs(w)) + 2 * UNIT * np.abs(z)
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    s = e.sum(1, keepdims=True)
    share = np.where(counted, share, 0.0)[:, None]
    worst = z_off.max(1, keepdims=True)
    out = {"loss": np.where(counted, np.log(s)[:, 0] - (z - m)[rows, at], 0.0)}
    off = {"loss": np.where(counted, 2 * worst[:, 0] + UNIT * (16 + 2 * np.abs((z - m)[rows, at]) + np.abs(out["loss"])), 0.0)}
    p = e / s
    dz = p * share
    p_off = 2 * worst + UNIT * (16 + 2 * (m - z))
    dz_off = np.abs(dz) * p_off
    rest = e.copy()
    rest[rows, at] = 0
    others = rest.sum(1) / s[:, 0]
    dz[rows, at] = -share[:, 0] * others
    # The others' sum is the difference of two sums of doubles, each of which rounds by 2^-53 of the whole at each addition.
    doubles = w.shape[1] * 2.0 ** -52
    dz_off[rows, at] = np.abs(share[:, 0]) * (others * (2 * worst[:, 0] + UNIT * (16 + 2 * np.abs((m - z) * p).sum(1))) + doubles)
    out["dx"], out["dw"], out["db"] = dz @ w.T, x.T @ dz, dz.sum(0)
    a, aw = np.abs(dz), np.abs(w)
    off["dx"] = dz_off @ aw.T + walk(w.shape[1]) * (a @ aw.T)
    off["dw"] = np.abs(x).T @ dz_off + walk(len(x)) * (np.abs(x).T @ a)
    off["db"] = dz_off.sum(0) + walk(len(x)) * a.sum(0)
    return out, off


def problem(rows, width, classes, seed=0, left_out=0.2, sure=4.0, bias=True):
    rng = np.random.default_rng(seed + rows + 31 * width + 1009 * classes)
    w = (rng.standard_normal((width, classes)) / np.sqrt(width)).astype(np.float32)
    t = rng.integers(0, classes, rows)
    x = (rng.standard_normal((rows, width)) + sure * rng.random((rows, 1)) * w[:, t].T).astype(np.float32)
    b = (0.5 * rng.standard_normal(classes)).astype(np.float32) if bias else None
    t = np.where(rng.random(rows) < left_out, -1, t)
    return x, w, t, b


def close(got, want, off):
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= off + 1e-37).all()


def run(x, w, t, b, device, reduction="mean", dy=None, host=False):
    leaf = lambda v: None if v is None else vc.Tensor(v, requires_grad=True, device=device)
    tx, tw, tb = leaf(x), leaf(w), leaf(b)
    targets = t if host else vc.Tensor(t.astype(np.float32), device=device)
    loss = vc.linear_cross_entropy(tx, tw, targets, bias=tb, reduction=reduction)
    if reduction == "mean":
        loss.backward()
    else:
        loss.backward(vc.Tensor(dy, device=device))
    shaped = lambda v: None if v is None else v.grad.numpy().reshape(v.shape)
    value = loss.item() if reduction == "mean" else loss.numpy()
    return value, shaped(tx), shaped(tw), shaped(tb)


SIZES = [(1, 1, 1), (1, 1, 2), (3, 5, 2), (1, 64, 10), (7, 64, 10), (64, 16, 256), (65, 33, 129), (33, 130, 257), (130, 96, 1000),
         (257, 128, 2049), (64, 511, 4099), (5, 300, 20001)]
# Larger ones of either side of whole tiles and lines, products that are packed (a fifth of the rows left out), and rows in more
# pieces than one of either route.
LARGE = [(1000, 96, 3001), (40, 700, 12000), (700, 1030, 400), (256, 1024, 1024), (999, 515, 10007), (2049, 1030, 1537),
         (513, 1030, 6007), (4099, 515, 2051), (257, 2050, 8200), (70000, 64, 515)]
CASES = [(*s, "cpu") for s in SIZES + LARGE[:3]] + [pytest.param(*s, "hip", marks=pytest.mark.gpu) for s in SIZES + LARGE]


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("rows,width,classes,device", CASES)
def test_mean(rows, width, classes, bias, device):
    x, w, t, b = problem(rows, width, classes, bias=bias)
    loss, dx, dw, db = run(x, w, t, b, device, host=rows % 2 == 0)
    number = max(1, (t >= 0).sum())
    want, off = exact(x, w, t, b, 1 / number)
    close(loss, want["loss"].sum() / number, off["loss"].sum() / number + 4 * UNIT * want["loss"].sum() / number)
    close(dx, want["dx"], off["dx"])
    close(dw, want["dw"], off["dw"])
    if bias:
        close(db, want["db"], off["db"])
    assert (dx[t < 0] == 0).all()


@pytest.mark.parametrize("rows,width,classes,device", CASES)
def test_none(rows, width, classes, device):
    x, w, t, b = problem(rows, width, classes, seed=1)
    dy = np.random.default_rng(rows).standard_normal(rows).astype(np.float32)
    loss, dx, dw, db = run(x, w, t, b, device, "none", dy)
    want, off = exact(x, w, t, b, dy.astype(np.float64))
    for got, name in ((loss, "loss"), (dx, "dx"), (dw, "dw"), (db, "db")):
        close(got, want[name], off[name])
    assert (loss[t < 0] == 0).all() and (dx[t < 0] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,width,classes", [(9, 20, 30), (300, 64, 3000), (900, 516, 10008)])
def test_left_out_rows_may_hold_anything(rows, width, classes, reduction, device):
    x, w, t, b = problem(rows, width, classes, seed=2, left_out=0.5)
    t[0] = -1
    dirty = x.copy()
    dirty[t < 0] = np.nan
    dirty[0] = np.inf
    dy = np.random.default_rng(7).random(rows).astype(np.float32)
    dirty_dy = np.where(t < 0, np.float32(np.nan), dy)
    clean, again = run(x, w, t, b, device, reduction, dy), run(dirty, w, t, b, device, reduction, dirty_dy)
    for a, c in zip(clean, again):
        np.testing.assert_array_equal(a, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(5, 6, 7), (260, 64, 2100), (900, 516, 10008)])
def test_no_row_counts(rows, width, classes, device):
    x, w, t, b = problem(rows, width, classes)
    loss, dx, dw, db = run(x, w, np.full(rows, -1), b, device)
    assert loss == 0 and (dx == 0).all() and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(300, 70, 90), (1100, 300, 9000)])
def test_the_largest_value_of_a_row_may_be_anywhere(rows, width, classes, device):
    """Rows of x and columns of the weight whose values are a thousandth of one of them, at every place of a row in turn."""
    x, w, t, b = problem(rows, width, classes, seed=3)
    x *= np.float32(1e-3)
    w *= np.float32(1e-3)
    x[np.arange(rows), np.arange(rows) % width] = 3.7
    w[(5 * np.arange(classes) + 3) % width, np.arange(classes)] = -1.9
    dy = np.random.default_rng(rows).random(rows).astype(np.float32)
    loss, dx, dw, db = run(x, w, t, b, device, "none", dy)
    want, off = exact(x, w, t, b, dy.astype(np.float64))
    for got, name in ((loss, "loss"), (dx, "dx"), (dw, "dw"), (db, "db")):
        close(got, want[name], off[name])


@pytest.mark.parametrize("rows,device", [(3, "cpu"), (9, "cpu"), pytest.param(3, "hip", marks=pytest.mark.gpu),
                                         pytest.param(33, "hip", marks=pytest.mark.gpu)])
def test_two_million_classes(rows, device):
    """More than the packed operands' offsets reach, and more logits than a piece of the other route holds; sums of millions
    of small products beside a large one."""
    x, w, t, b = problem(rows, 2, 2 ** 21 + 3, bias=False)
    loss, dx, dw, _ = run(x, w, t, b, device)
    number = (t >= 0).sum()
    want, off = exact(x, w, t, b, 1 / number)
    close(loss, want["loss"].sum() / number, off["loss"].sum() / number + 4 * UNIT * want["loss"].sum() / number)
    close(dx, want["dx"], off["dx"])
    close(dw, want["dw"], off["dw"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("width,classes", [(1, 1), (15, 127), (17, 129), (130, 128), (257, 1001)])
def test_scores_of_a_few_rows(rows, width, classes, device):
    """Without gradients, and of rows some of which are left out."""
    x, w, t, b = problem(rows, width, classes)
    t[0] = classes - 1
    tensors = [vc.Tensor(v, device=device) for v in (x, w)]
    bias = vc.Tensor(b, device=device)
    want, off = exact(x, w, t, b, 1.0)
    each = vc.linear_cross_entropy(*tensors, t, bias=bias, reduction="none")
    assert not each.requires_grad
    close(each.numpy(), want["loss"], off["loss"])
    number = (t >= 0).sum()
    mean = vc.linear_cross_entropy(*tensors, t, bias=bias).item()
    close(mean, want["loss"].sum() / number, off["loss"].sum() / number + 4 * UNIT * want["loss"].sum() / number)


@pytest.mark.parametrize("device", DEVICES)
def test_numbers_that_are_no_class(device):
    x, w, _, b = problem(8, 12, 10, left_out=0)
    t = np.array([3, -1, 10, 2.5, np.nan, np.inf, -0.0, 9], np.float32)
    loss = vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w, t)), bias=vc.Tensor(b, device=device), reduction="none")
    want, off = exact(x, w, np.array([3, -1, -1, -1, -1, -1, 0, 9]), b, 1.0)
    close(loss.numpy(), want["loss"], off["loss"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(6, 24, 50), (300, 24, 2500), (1100, 300, 9000)])
def test_classes_without_a_chance(rows, width, classes, device):
    """A bias of minus infinity, and the type's lowest value, take a class out; a target among them loses everything."""
    for lowest in (-np.inf, np.finfo(np.float32).min):
        x, w, t, b = problem(rows, width, classes, left_out=0)
        out = np.arange(0, classes, 3)
        t = np.where(t % 3 == 0, (t + 1) % classes, t)
        t = np.where(t % 3 == 0, 1, t)
        b[out] = lowest
        loss, dx, dw, db = run(x, w, t, b, device)
        keep = np.setdiff1d(np.arange(classes), out)
        want, off = exact(x, w[:, keep], np.searchsorted(keep, t), b[keep], 1 / rows)
        close(loss, want["loss"].mean(), off["loss"].mean() + 4 * UNIT * want["loss"].mean())
        close(dx, want["dx"], off["dx"])
        close(dw[:, keep], want["dw"], off["dw"])
        assert (dw[:, out] == 0).all() and (db[out] == 0).all()
        t[0] = 0
        each = vc.linear_cross_entropy(vc.Tensor(x, device=device), vc.Tensor(w, device=device), t, bias=vc.Tensor(b, device=device),
                                       reduction="none").numpy()
        assert each[0] > 1e38 and np.isfinite(each[1:]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(70, 16, 40), (70, 16, 3000), (1100, 300, 9000)])
def test_sure_rows_keep_their_small_gradients(rows, width, classes, device):
    """A target of probability 1 - 1e-9: one minus a float32 share would leave nothing of the gradient."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((rows, width)).astype(np.float32)
    w = np.zeros((width, classes), np.float32)
    t = rng.integers(0, classes, rows)
    b = np.full(classes, -20.0, np.float32)
    b[5] = 8.0
    t[:] = 5
    loss, dx, dw, db = run(x, w, t, b, device)
    want, off = exact(x, w, t, b, 1 / rows)
    assert 0 < -want["db"][5] < 1e-7
    close(dw, want["dw"], off["dw"])
    close(db, want["db"], off["db"])
    assert abs(loss - want["loss"].mean()) <= off["loss"].mean()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(4, 16, 30), (19, 16, 30), (260, 16, 2100), (1100, 300, 9000)])
def test_a_row_of_nan_gives_nan(rows, width, classes, device):
    x, w, t, b = problem(rows, width, classes, left_out=0)
    x[1, 3] = np.nan
    each = vc.linear_cross_entropy(vc.Tensor(x, device=device), vc.Tensor(w, device=device), t, reduction="none").numpy()
    assert np.isnan(each[1]) and np.isfinite(np.delete(each, 1)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wanted", ["x", "weight", "bias"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,width,classes", [(12, 40, 37), (270, 40, 2300), (1500, 1026, 10010)])
def test_one_gradient_alone(rows, width, classes, reduction, wanted, device):
    x, w, t, b = problem(rows, width, classes)
    leaf = lambda v, name: vc.Tensor(v, requires_grad=name == wanted, device=device)
    tensors = {"x": leaf(x, "x"), "weight": leaf(w, "weight"), "bias": leaf(b, "bias")}
    loss = vc.linear_cross_entropy(tensors["x"], tensors["weight"], t, bias=tensors["bias"], reduction=reduction)
    loss.sum().backward()
    assert [n for n in tensors if tensors[n].grad is not None] == [wanted]
    want, off = exact(x, w, t, b, 1.0 if reduction == "none" else 1 / (t >= 0).sum())
    name = {"x": "dx", "weight": "dw", "bias": "db"}[wanted]
    close(tensors[wanted].grad.numpy(), want[name], off[name])


@pytest.mark.parametrize("device", DEVICES)
def test_upstream_gradients_scale_and_add_up(device):
    """Half the loss, then the graph a second time, without the first pass's gradients being touched."""
    x, w, t, b = problem(20, 10, 15)
    tx, tw = (vc.Tensor(v, requires_grad=True, device=device) for v in (x, w))
    loss = vc.linear_cross_entropy(tx, tw, t)
    loss.backward()
    once = tx.grad.numpy().copy(), tw.grad.numpy().copy()
    (loss * 0.5).backward()
    # A product with a power of two and one sum.
    np.testing.assert_allclose(tx.grad.numpy(), 1.5 * once[0], rtol=2 * UNIT, atol=0)
    np.testing.assert_allclose(tw.grad.numpy(), 1.5 * once[1], rtol=2 * UNIT, atol=0)
    tx.zero_grad()
    vc.sgd_step([tw], 0.1)  # the mean loss's gradients are those of the values that it was computed from
    loss.backward()
    np.testing.assert_array_equal(tx.grad.numpy(), once[0])


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_given_away_may_be_written(device):
    """What a first pass stores may be written to in place: a later pass through the same graph gives the same again."""
    x, w, t, b = problem(20, 10, 15)
    tx, tw = (vc.Tensor(v, requires_grad=True, device=device) for v in (x, w))
    loss = vc.linear_cross_entropy(tx, tw, t)
    loss.backward()
    once = tx.grad.numpy().copy(), tw.grad.numpy().copy()
    held = tw.grad
    held.requires_grad = True
    held.sum().backward()
    vc.sgd_step([held], 1.0)  # subtracts one everywhere
    np.testing.assert_array_equal(held.numpy(), once[1] - 1)
    tx.zero_grad(), tw.zero_grad()
    loss.backward()
    np.testing.assert_array_equal(tx.grad.numpy(), once[0])
    np.testing.assert_array_equal(tw.grad.numpy(), once[1])


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    x, w, t, b = problem(4, 6, 9)
    _, dx, dw, db = run(x, w, t, b, device)
    number = (t >= 0).sum()
    value = lambda *a: exact(a[0], a[1], t, a[2], 1.0)[0]["loss"].sum() / number
    step = 1e-5
    for which, got in ((0, dx), (1, dw), (2, db)):
        for i in np.ndindex(got.shape):
            ends = []
            for sign in (1, -1):
                args = [v.astype(np.float64) for v in (x, w, b)]
                args[which][i] += sign * step
                ends.append(value(*args))
            # The third difference of a function of order one, and float32.
            assert abs((ends[0] - ends[1]) / (2 * step) - got[i]) <= 2e-6


@pytest.mark.parametrize("device", DEVICES)
def test_the_same_as_the_logits_loss(device):
    x, w, t, b = problem(50, 30, 40, left_out=0)
    tx, tw, tb = (vc.Tensor(v, requires_grad=True, device=device) for v in (x, w, b))
    vc.cross_entropy(tx @ tw + tb, t).backward()
    _, dx, dw, db = run(x, w, t, b, device)
    _, off = exact(x, w, t, b, 1 / 50)
    assert (np.abs(tx.grad.numpy() - dx) <= 2 * off["dx"] + 8 * UNIT * np.abs(w).max()).all()
    assert (np.abs(tw.grad.numpy() - dw) <= 2 * off["dw"] + 8 * UNIT * np.abs(x).max()).all()
    assert (np.abs(tb.grad.numpy() - db) <= 2 * off["db"] + 8 * UNIT).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(40, 50, 60), (300, 200, 2222), (900, 516, 10008)])
def test_repeats_are_equal(rows, width, classes, device):
    x, w, t, b = problem(rows, width, classes)
    runs = [run(x, w, t, b, device) for _ in range(3)]
    for again in runs[1:]:
        for a, c in zip(runs[0], again):
            np.testing.assert_array_equal(a, c)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    t = lambda *shape: vc.Tensor(np.zeros(shape, np.float32), device=device)
    loss = vc.linear_cross_entropy
    for bad in (lambda: loss(t(3), t(3, 4), [0, 0, 0]), lambda: loss(t(3, 4), t(4), [0, 0, 0]), lambda: loss(t(3, 4), t(5, 6), [0, 0, 0]),
                lambda: loss(t(3, 4), t(4, 6), [0, 0]), lambda: loss(t(3, 4), t(4, 6), t(4)), lambda: loss(t(3, 4), t(4, 6), t(3, 1)),
                lambda: loss(t(3, 4), t(4, 6), [0, 0, 0], bias=t(5)), lambda: loss(t(3, 4), t(4, 6), [0, 0, 0], bias=t(1, 6)),
                lambda: loss(t(3, 4), t(4, 6), [0, 0, 0], reduction="sum"), lambda: loss(t(3, 0), t(0, 6), [0, 0, 0]),
                lambda: loss(t(3, 4), t(4, 0), [0, 0, 0]), lambda: loss(t(0, 4), t(4, 6), []),
                lambda: loss(t(3, 4), t(4, 6), np.zeros((3, 1), int))):
        with pytest.raises(ValueError):
            bad()
    for bad in ([0, 6, 0], [0, -2, 0], np.array([0, 1, 6])):
        with pytest.raises(IndexError):
            loss(t(3, 4), t(4, 6), bad)
    assert tuple(loss(t(0, 4), t(4, 6), [], reduction="none").shape) == (0,)
    if device == "hip":
        with pytest.raises(ValueError, match="expected hip"):
            loss(t(3, 4), vc.Tensor(np.zeros((4, 6), np.float32)), [0, 0, 0])
        with pytest.raises(ValueError, match="expected hip"):
            loss(t(3, 4), t(4, 6), vc.Tensor(np.zeros(3, np.float32)))


@pytest.mark.parametrize("device", DEVICES)
def test_an_operand_changed_in_place_is_noticed(device):
    x, w, t, _ = problem(6, 5, 4, left_out=0)
    tx, tw = (vc.Tensor(v, requires_grad=True, device=device) for v in (x, w))
    each = vc.linear_cross_entropy(tx, tw, t, reduction="none").sum()
    tw.sum().backward()
    vc.sgd_step([tw], 0.5)
    with pytest.raises(RuntimeError):
        each.backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(24, 16, 20), (300, 96, 2200)])
def test_a_block_and_its_loss(rows, width, classes, device):
    """Normalise, a linear layer, drop out onto the stream, normalise again, the loss: a step of all three together, the
    gradients by differences along random directions of the same program in float64."""
    from test_dropout import words
    rng = np.random.default_rng(rows)
    values = {"x": rng.standard_normal((rows, width)), "w": rng.standard_normal((width, width)) / np.sqrt(width),
              "g": 1 + 0.1 * rng.standard_normal(width), "head": rng.standard_normal((width, classes)) / np.sqrt(width)}
    values = {n: v.astype(np.float32) for n, v in values.items()}
    t = np.where(rng.random(rows) < 0.2, -1, rng.integers(0, classes, rows))
    v = {n: vc.Tensor(a, requires_grad=True, device=device) for n, a in values.items()}
    h = vc.dropout(vc.layer_norm(v["x"], v["g"]) @ v["w"], 0.25, 17, stream=3, residual=v["x"])
    loss = vc.linear_cross_entropy(vc.layer_norm(h), v["head"], t)
    loss.backward()
    factor = (words(rows * width, 17, 3) >= 2 ** 30).reshape(rows, width) / 0.75

    def program(a):
        norm = lambda z: (z - z.mean(1, keepdims=True)) / np.sqrt(z.var(1, keepdims=True) + float(np.float32(1e-5)))
        z = norm(a["x"] + factor * ((norm(a["x"]) * a["g"]) @ a["w"])) @ a["head"]
        z = z - z.max(1, keepdims=True)
        each = np.log(np.exp(z).sum(1)) - z[np.arange(rows), np.where(t < 0, 0, t)]
        return each[t >= 0].sum() / max(1, (t >= 0).sum())

    double = {n: a.astype(np.float64) for n, a in values.items()}
    # A dozen roundings of values of a few units on the way, and the logarithm.
    assert abs(loss.item() - program(double)) <= 64 * UNIT * (1 + program(double))
    for n in values:
        direction = rng.standard_normal(values[n].shape)
        step = 1e-5
        ends = [program(dict(double, **{n: double[n] + sign * step * direction})) for sign in (1, -1)]
        slope, got = (ends[0] - ends[1]) / (2 * step), (v[n].grad.numpy() * direction).sum()
        size = np.linalg.norm(v[n].grad.numpy()) * np.linalg.norm(direction)
        assert abs(slope - got) <= 1e-6 * size + 1e-7
