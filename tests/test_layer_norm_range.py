"""Layer normalisation of rows near the ends of float32's range, alike for rows of every length and on both
devices."""

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
def test_one_row_does_not_change_another(device):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 300)).astype(np.float32)
    alone = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    x[1] *= np.float32(1e30)
    x[4] *= np.float32(1e-36)
    y = vc.layer_norm(vc.Tensor(x, device=device)).numpy()
    np.testing.assert_array_equal(y[[0, 2, 3, 5]], alone[[0, 2, 3, 5]])
