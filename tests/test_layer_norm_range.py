"""Layer normalisation of rows near the ends of float32's range, alike for rows of every length and on both devices, and sums
over very many rows."""

import numpy as np
import pytest

import vectorcore_amd as vc
from test_layer_norm import DEVICES, UNIT, check, grad_of, leaf

WIDTHS = [4, 64, 515, 4096, 9000, 16384, 16385]


def step(x, dy, device, eps, affine=True):
    width = x.shape[1]
    rng = np.random.default_rng(width)
    w = (1 + 0.2 * rng.standard_normal(width)).astype(np.float32) if affine else None
    b = rng.standard_normal(width).astype(np.float32) if affine else None
    tx, tw, tb = leaf(x, device), leaf(w, device), leaf(b, device)
    y = vc.layer_norm(tx, tw, tb, eps=eps)
    y.backward(vc.Tensor(dy, device=device))
    check(x, w, b, float(np.float32(eps)), dy, y.numpy(), grad_of(tx), grad_of(tw), grad_of(tb))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("size,eps", [(1e19, 1e-5), (1e20, 1e-5), (1e30, 1e-5), (1e37, 1e-5), (1e30, 0.0), (1e-22, 0.0), (1e-25, 0.0),
                                      (1e-35, 0.0), (1e-25, 1e-5)])
@pytest.mark.parametrize("width", WIDTHS)
def test_rows_of_any_size(width, size, eps, device):
    """Deviations whose squares no float holds; the gradient of a row is as small as the row is large, so dy is of its size."""
    rng = np.random.default_rng(width)
    x = (size * (rng.standard_normal((3, width)) + rng.standard_normal((3, 1)))).astype(np.float32)
    dy = (min(size, 1e33) * rng.standard_normal((3, width))).astype(np.float32)
    step(x, dy, device, eps)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", WIDTHS)
def test_rows_of_the_largest_floats(width, device):
    """Both signs of values whose differences no float holds, and one sign, whose sums none does."""
    rng = np.random.default_rng(width)
    x = np.stack([np.where(rng.random(width) < 0.5, -3.2e38, 3.2e38), 3e38 + 1e37 * rng.random(width), 3e38 * rng.random(width)])
    x[0, :2] = 3.2e38, -3.2e38
    dy = (1e33 * rng.standard_normal((3, width))).astype(np.float32)
    step(x.astype(np.float32), dy, device, 1e-5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", WIDTHS)
def test_upstream_gradients_whose_sums_no_float_holds(width, device):
    rng = np.random.default_rng(width)
    x = rng.standard_normal((2, width)).astype(np.float32)
    dy = (1e38 * (0.5 + 0.2 * rng.random((2, width)))).astype(np.float32)
    step(x, dy, device, 1e-5, affine=False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("eps", [1e-5, 1e-30])
@pytest.mark.parametrize("width", WIDTHS + [49, 98, 103, 107, 161, 1000, 3000])  # n (1 / n) is not one for some of them
def test_equal_values_of_any_size_are_zeros(width, eps, device):
    """Their mean is exact, so that nothing but eps is left of the variance, and the gradient is one over its root."""
    values = np.float32([1e7, -1.2345678e8, 3e20, -1.1e38, 3.3e38, 1e-7, 1e-25, -1e-38, 0])
    x = np.repeat(values[:, None], width, 1)
    dy = np.random.default_rng(width).standard_normal(x.shape).astype(np.float32)
    tx = leaf(x, device)
    y = vc.layer_norm(tx, eps=eps)
    y.backward(vc.Tensor(dy, device=device))
    assert (y.numpy() == 0).all()
    d = dy - dy.astype(np.float64).mean(1, keepdims=True)
    root = np.sqrt(float(np.float32(eps)))
    # The mean of dy by sums of at most 32 roundings of the mean magnitude, and roundings of the difference and the products.
    assert (np.abs(grad_of(tx) - d / root) <= UNIT / root * (8 * np.abs(d) + 40 * np.abs(dy).mean(1, keepdims=True))).all()


@pytest.mark.parametrize("device", DEVICES)
def test_one_row_does_not_change_another(device):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 300)).astype(np.float32)
    alone = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    x[1] *= np.float32(1e30)
    x[4] *= np.float32(1e-36)
    y = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    np.testing.assert_array_equal(y[[0, 2, 3, 5]], alone[[0, 2, 3, 5]])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(2 ** 21 + 3, 500), (2 ** 19 + 1, 4000), (2 ** 24 + 5, 12)])
def test_sums_over_many_equal_rows(rows, width):
    """Equal terms, whose roundings do not cancel: of a float32 sum of n of them each addition may lose half a step of it, UNIT
    n / 2 of the whole. Sixty-four are added so, the rest in double; and a product and a deviation's roundings for the weight."""
    rng = np.random.default_rng(width)
    row, d = rng.standard_normal(width).astype(np.float32), (1 + rng.random(width)).astype(np.float32)
    ones = vc.Tensor(np.ones((rows, 1), np.float32), device="hip")
    x, dy = (ones * vc.Tensor(v, device="hip") for v in (row, d))
    w, b = (leaf(np.ones(width, np.float32), "hip") for _ in range(2))
    vc.layer_norm(x, w, b).backward(dy)
    h = row.astype(np.float64) - row.astype(np.float64).mean()
    h /= np.sqrt((h * h).mean() + float(np.float32(1e-5)))
    assert (np.abs(grad_of(b) / (rows * d.astype(np.float64)) - 1) <= 34 * UNIT).all()
    assert (np.abs(grad_of(w) - rows * h * d) <= rows * d * UNIT * (42 * np.abs(h) + 8)).all()
