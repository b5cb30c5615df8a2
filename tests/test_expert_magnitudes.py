"""Expert products of values next to float32's least: what float32 holds from 2^-110 on, and an error of half of
bfloat16's least step, 2^-134, below."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [2, 70, 300])
@pytest.mark.parametrize("least", [100, 110, 116, 120, 126])
def test_small_values_beside_large_ones(least, rows, device):
    """Rows of about 2^-least and a matrix of about 2^100: a linear map and the gradient of its input."""
    rng = np.random.default_rng(least)
    width, columns = 96, 80
    signed = lambda *s: rng.uniform(1, 2, s) * rng.choice([-1, 1], s)
    x, w, g = (v.astype(np.float32) for v in (np.ldexp(signed(rows, width), -least), np.ldexp(signed(1, width, columns), 100),
                                              np.ldexp(signed(rows, columns), -least)))
    plan = vc.ExpertPlan(vc.Tensor(np.zeros((rows, 1), np.float32), device=device), 1)
    tx, tw = (vc.Tensor(v, requires_grad=True, device=device) for v in (x, w))
    y = vc.expert_linear(tx, tw, plan)
    y.backward(vc.Tensor(g, device=device))
    step = 2.0 ** -134 if least > 110 and device == "hip" else 0.0
    for got, a, b in ((y, x, w[0]), (tx.grad, g, w[0].T)):
        a, b = a.astype(np.float64), b.astype(np.float64)
        # A sum of k products in float32 (with its own few roundings), and the small factors' steps.
        most = ((a.shape[1] + 8) * UNIT * np.abs(a) + step) @ np.abs(b)
        assert (np.abs(got.numpy() - a @ b) <= most).all()
