"""Layer normalisation against its definition in float64: row lengths on either side of every kernel's reach, rows far from
zero, constant rows, infinities and NaN, gradients (also against differences), views, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


def exact(x, w, b, eps, dy=None):
    x = x.astype(np.float64)
    w = np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    b = np.zeros(x.shape[-1]) if b is None else b.astype(np.float64)
    c = x - x.mean(-1, keepdims=True)
    r = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    h = c * r
    out = {"y": h * w + b, "h": h, "r": r, "w": w, "b": b}
    if dy is not None:
        d = dy.astype(np.float64) * w
        out["dx"] = r * (d - d.mean(-1, keepdims=True) - h * (d * h).mean(-1, keepdims=True))
        out["dw"], out["db"] = (dy * h).sum(0), dy.astype(np.float64).sum(0)
    return out


def check(x, w, b, eps, dy, y, dx, dw, db):
    """Sums of n values go by lanes of at most 16 and a tree of at most 16 additions: 32 roundings of the mean magnitude. A
    deviation is rounded twice and off by its mean's error, the scale by half its sum's, and each product once."""
    e = exact(x, w, b, eps, dy)
    h, r, d = np.abs(e["h"]), e["r"], np.abs(dy * e["w"])
    h_off = 48 * UNIT * (h + 1)
    assert (np.abs(y - e["y"]) <= h_off * np.abs(e["w"]) + 4 * UNIT * (np.abs(e["y"]) + np.abs(e["b"])) + 1e-37).all()
    mean = lambda v: v.mean(-1, keepdims=True)
    if dx is not None:
        off = 4 * d + 40 * mean(d) + 96 * (h + 1) * mean(d * (h + 1))
        assert (np.abs(dx - e["dx"]) <= UNIT * r * off + 24 * UNIT * np.abs(e["dx"]) + 1e-37).all()
    # A thread adds its rows one after another in float32, then doubles: at most 64 of the tested sizes.
    if dw is not None:
        assert (np.abs(dw - e["dw"]) <= UNIT * 112 * (np.abs(dy) * (h + 1)).sum(0) + 1e-37).all()
    if db is not None:
        assert (np.abs(db - e["db"]) <= UNIT * 64 * np.abs(dy).sum(0) + 1e-37).all()


def leaf(values, device, grad=True):
    return None if values is None else vc.Tensor(values, requires_grad=grad, device=device)


def grad_of(t):
    return None if t is None else t.grad.numpy().reshape(t.shape)


WIDTHS = [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 128, 129, 255, 256, 257, 511, 512, 513, 767, 769, 1023, 1024, 1025, 2047, 2049, 3071,
          4095, 4096, 4097, 8191, 8193, 12289, 16383, 16384, 16385, 40001]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("affine", ["both", "weight", "bias", "none"])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, affine, device):
    rng = np.random.default_rng(width)
    rows = 3 if width > 2000 else 37
    x = (rng.standard_normal((rows, width)) * (1 + 3 * rng.random((rows, 1))) + rng.standard_normal((rows, 1))).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32) if affine in ("both", "weight") else None
    b = rng.standard_normal(width).astype(np.float32) if affine in ("both", "bias") else None
    dy = rng.standard_normal((rows, width)).astype(np.float32)
    tx, tw, tb = leaf(x, device), leaf(w, device), leaf(b, device)
    y = vc.layer_norm(tx, tw, tb, eps=1e-5)
    y.backward(vc.Tensor(dy, device=device))
    eps = float(np.float32(1e-5))
    check(x, w, b, eps, dy, y.numpy(), grad_of(tx), grad_of(tw), grad_of(tb))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [0, 1, 2, 511, 512, 513, 4097])
@pytest.mark.parametrize("width", [3, 64, 300])
def test_row_counts(rows, width, device):
    rng = np.random.default_rng(rows + width)
    x, dy = (rng.standard_normal((rows, width)).astype(np.float32) for _ in range(2))
    w, b = (rng.standard_normal(width).astype(np.float32) for _ in range(2))
    tx, tw, tb = leaf(x, device), leaf(w, device), leaf(b, device)
    y = vc.layer_norm(tx, tw, tb)
    y.backward(vc.Tensor(dy, device=device))
    shape = lambda t: t.numpy().reshape(t.shape)
    check(x, w, b, float(np.float32(1e-5)), dy, shape(y), grad_of(tx), grad_of(tw), grad_of(tb))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [33, 700, 5000, 20000])
@pytest.mark.parametrize("far", [1e3, -1e6])
def test_rows_far_from_zero(width, far, device):
    """A mean of a million and a deviation of one: the mean of the floats is what counts, to more bits than a float has."""
    rng = np.random.default_rng(5)
    x = (far + rng.standard_normal((4, width))).astype(np.float32)
    dy = rng.standard_normal((4, width)).astype(np.float32)
    tx = leaf(x, device)
    y = vc.layer_norm(tx, eps=1e-5)
    y.backward(vc.Tensor(dy, device=device))
    check(x, None, None, float(np.float32(1e-5)), dy, y.numpy(), grad_of(tx), None, None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [1, 7, 64, 1500, 9000, 17000])
def test_constant_rows_are_zeros(width, device):
    x = np.full((3, width), 0.1, np.float32)
    x[1], x[2] = 0.0, -12345.678
    b = np.linspace(-1, 1, width).astype(np.float32)
    y = vc.layer_norm(vc.Tensor(x, device=device), bias=vc.Tensor(b, device=device))
    # Deviations of a rounding's error, over sqrt(eps).
    np.testing.assert_allclose(y.numpy(), np.broadcast_to(b, (3, width)), atol=1e-37 + 4 * UNIT, rtol=0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [5, 64, 1500, 9000, 17000])
def test_infinities_and_nan_stay_in_their_row(width, device):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, width)).astype(np.float32)
    clean = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    x[1, width // 2], x[3, 0] = np.nan, np.inf
    y = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    assert np.isnan(y[[1, 3]]).all()
    np.testing.assert_array_equal(y[[0, 2, 4]], clean[[0, 2, 4]])


@pytest.mark.parametrize("device", DEVICES)
def test_axes_and_offsets(device):
    """The last of four axes, and the gradient that arrives through a reshape."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((2, 3, 4, 6)).astype(np.float32)
    dy = rng.standard_normal((24, 6)).astype(np.float32)
    tx = leaf(x, device)
    y = vc.layer_norm(tx)
    assert tuple(y.shape) == (2, 3, 4, 6)
    y.reshape((24, 6)).backward(vc.Tensor(dy, device=device))
    check(x.reshape(24, 6), None, None, float(np.float32(1e-5)), dy, y.numpy().reshape(24, 6), grad_of(tx).reshape(24, 6), None, None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("wanted", ["x", "weight", "bias"])
@pytest.mark.parametrize("width", [48, 6000, 14000, 18000])
def test_one_gradient_alone(width, wanted, device):
    rng = np.random.default_rng(width)
    x, dy = (rng.standard_normal((9, width)).astype(np.float32) for _ in range(2))
    w, b = (rng.standard_normal(width).astype(np.float32) for _ in range(2))
    t = {"x": leaf(x, device, wanted == "x"), "weight": leaf(w, device, wanted == "weight"), "bias": leaf(b, device, wanted == "bias")}
    y = vc.layer_norm(t["x"], t["weight"], t["bias"])
    y.backward(vc.Tensor(dy, device=device))
    assert [n for n in t if t[n].grad is not None] == [wanted]
    got = {n: grad_of(t[n]) if n == wanted else None for n in t}
    check(x, w, b, float(np.float32(1e-5)), dy, y.numpy(), got["x"], got["weight"], got["bias"])


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((3, 11)), rng.standard_normal((3, 11)).astype(np.float32)
    w, b = (rng.standard_normal(11).astype(np.float32) for _ in range(2))
    tx = leaf(x.astype(np.float32), device)
    vc.layer_norm(tx, leaf(w, device), leaf(b, device), eps=0.25).backward(vc.Tensor(dy, device=device))
    x = x.astype(np.float32).astype(np.float64)
    step = 1e-5
    for i in np.ndindex(3, 11):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        slope = ((exact(up, w, b, 0.25)["y"] - exact(down, w, b, 0.25)["y"]) * dy).sum() / (2 * step)
        assert abs(slope - grad_of(tx)[i]) <= 1e-5  # the third difference of a function of order one, and float32


@pytest.mark.parametrize("device", DEVICES)
def test_no_gradient_and_repeats(device):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((700, 515)).astype(np.float32)
    w = rng.standard_normal(515).astype(np.float32)
    assert not vc.layer_norm(vc.Tensor(x, device=device)).requires_grad
    runs = []
    for _ in range(3):
        tx, tw = leaf(x, device), leaf(w, device)
        y = vc.layer_norm(tx, tw)
        y.backward(y.detach())
        runs.append((y.numpy(), grad_of(tx), grad_of(tw)))
    for again in runs[1:]:
        for a, b in zip(runs[0], again):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    t = lambda *shape: vc.Tensor(np.ones(shape, np.float32), device=device)
    other = vc.Tensor(np.ones(4, np.float32), device="cpu" if device == "hip" else "cpu")
    for bad in (lambda: vc.layer_norm(vc.Tensor(1.0, device=device)), lambda: vc.layer_norm(t(3, 0)),
                lambda: vc.layer_norm(t(3, 4), t(3)), lambda: vc.layer_norm(t(3, 4), t(1, 4)), lambda: vc.layer_norm(t(3, 4), None, t(5)),
                lambda: vc.layer_norm(t(3, 4), eps=-1.0), lambda: vc.layer_norm(t(3, 4), eps=float("nan")),
                lambda: vc.layer_norm(t(3, 4), eps=float("inf"))):
        with pytest.raises(ValueError):
            bad()
    if device == "hip":
        with pytest.raises(ValueError, match="expected hip"):
            vc.layer_norm(t(3, 4), other)


@pytest.mark.parametrize("device", DEVICES)
def test_an_input_changed_in_place_is_noticed(device):
    x = vc.Tensor(np.ones((2, 4), np.float32), requires_grad=True, device=device)
    y = vc.layer_norm(x).sum()
    x.sum().backward()
    vc.sgd_step([x], 0.5)
    with pytest.raises(RuntimeError):
        y.backward()
