"""Calls of the layers' operators that their signatures allow: one tensor in two places, targets of other types, rows of one
value, upstream gradients of zero."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [4, 33, 700])
def test_one_tensor_as_rows_and_weight(n, device):
    rng = np.random.default_rng(n)
    a = (rng.standard_normal((n, n)) / np.sqrt(n)).astype(np.float32)
    q = vc.Tensor(a, requires_grad=True, device=device)
    vc.linear_cross_entropy(q, q, np.arange(n)).backward()
    d = a.astype(np.float64)
    z = d @ d
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    dz = (p - np.eye(n)) / n
    # Of both products' terms, a rounding of the logits' (2 z, and of their n terms 4 sqrt(n) at eight deviations) and of the sum.
    worst = UNIT * ((8 + 4 * np.sqrt(n)) * (np.abs(d) @ np.abs(d)).max() + 2 * np.abs(z).max())
    size = (np.abs(dz) + p / n) @ np.abs(d.T) + np.abs(d.T) @ (np.abs(dz) + p / n)
    off = size * (2 * worst + UNIT * (32 + 4 * np.sqrt(n)))
    assert (np.abs(q.grad.numpy() - (dz @ d.T + d.T @ dz)) <= off).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_tensor_as_weight_and_bias_and_row(device):
    rng = np.random.default_rng(5)
    a = rng.standard_normal(70).astype(np.float32)
    v = vc.Tensor(a, requires_grad=True, device=device)
    y = vc.layer_norm(v, v, v)
    y.sum().backward()
    d = a.astype(np.float64)
    scale = 1 / np.sqrt(d.var() + float(np.float32(1e-5)))
    h = (d - d.mean()) * scale
    # Sums of 70 terms, a dozen roundings of values of at most 10 each way.
    off = UNIT * 32 * np.sqrt(70) * (1 + np.abs(d)) * (1 + np.abs(h))
    assert (np.abs(y.numpy() - (h * d + d)) <= off).all()
    assert (np.abs(v.grad.numpy() - (scale * (d - d.mean() - h * (d * h).mean()) + h + 1)) <= 4 * off * max(1, scale)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_targets_of_other_types(device):
    rng = np.random.default_rng(3)
    x, w = (vc.Tensor(rng.standard_normal(s).astype(np.float32), device=device) for s in ((3, 5), (5, 4)))
    loss = lambda t: vc.linear_cross_entropy(x, w, t, reduction="none").numpy()
    want = loss([0, 3, -1])
    for kind in (np.int8, np.int32, np.int64):
        np.testing.assert_array_equal(loss(np.array([0, 3, -1], kind)), want)
    np.testing.assert_array_equal(loss(np.array([9, 0, 9, 3, 9, -1])[1::2]), want)
    np.testing.assert_array_equal(loss(np.array([0, 3, 1], np.uint64)), loss([0, 3, 1]))
    np.testing.assert_array_equal(loss(vc.Tensor(np.float32([0, 3, np.nan]), device=device)), want)
    # An array of floats would lose its fractions and NaN; the largest uint64 is not -1.
    for bad in (np.float32([0, 3, 1]), np.array([0.5, 1, 2]), np.array([True, False, True]), np.array(["0", "1", "2"])):
        with pytest.raises(ValueError, match="integers"):
            loss(bad)
    with pytest.raises(IndexError):
        loss(np.array([0, 1, 2 ** 64 - 1], np.uint64))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", [(20, 24, 30), (999, 515, 4099)])
def test_upstream_gradients_of_zero(rows, width, classes, device):
    if device == "cpu" and rows > 100:
        rows, width, classes = 50, 40, 300
    rng = np.random.default_rng(rows)
    x, w = rng.standard_normal((rows, width)), rng.standard_normal((width, classes)) / np.sqrt(width)
    tx, tw = (vc.Tensor(v.astype(np.float32), requires_grad=True, device=device) for v in (x, w))
    t = rng.integers(0, classes, rows)
    vc.linear_cross_entropy(tx, tw, t, reduction="none").backward(vc.Tensor(np.zeros(rows, np.float32), device=device))
    assert (tx.grad.numpy() == 0).all() and (tw.grad.numpy() == 0).all()
    # One row alone has a share: the others' gradients are zero, the weight's those of a call with that row alone.
    tx, tw = (vc.Tensor(v.astype(np.float32), requires_grad=True, device=device) for v in (x, w))
    dy = np.zeros(rows, np.float32)
    dy[rows // 2] = 0.5
    vc.linear_cross_entropy(tx, tw, t, reduction="none").backward(vc.Tensor(dy, device=device))
    dx = tx.grad.numpy()
    row = rows // 2
    assert (np.delete(dx, row, 0) == 0).all() and (dx[row] != 0).any()
    p = np.float32(x[row]).astype(np.float64) @ np.float32(w).astype(np.float64)
    p = np.exp(p - p.max())
    p /= p.sum()
    p[t[row]] -= 1
    want = 0.5 * np.outer(np.float32(x[row]), p)
    # As the logits: of width terms 4 sqrt(width) roundings at eight deviations, and those of a handful of functions.
    z_off = UNIT * (8 + 4 * np.sqrt(width)) * (np.abs(x[row]) @ np.abs(w)).max()
    off = 0.5 * np.outer(np.abs(x[row]), np.abs(p) + UNIT) * (2 * z_off + 64 * UNIT)
    assert (np.abs(tw.grad.numpy() - want) <= off + 1e-12).all()


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_one_value(device):
    v = vc.Tensor(np.float32([[3], [-4], [0]]), requires_grad=True, device=device)
    w, b = (vc.Tensor(np.float32([u]), requires_grad=True, device=device) for u in (2.0, 0.25))
    y = vc.layer_norm(v, w, b)
    y.sum().backward()
    np.testing.assert_array_equal(y.numpy(), np.full((3, 1), 0.25, np.float32))
    np.testing.assert_array_equal(v.grad.numpy().reshape(-1), np.zeros(3, np.float32))
    assert w.grad.item() == 0 and b.grad.item() == 3
