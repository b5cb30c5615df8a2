"""Experts whose scores differ in no bit of 64, though their logits differ: equal ranks go to the lower index, also behind
equal logits."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]


def first_best(scores, top_k):
    return np.argsort(-scores, axis=1, kind="stable")[:, :top_k]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("top_k", [1, 2, 5])
@pytest.mark.parametrize("experts", [7, 30, 64, 200, 300])
def test_saturated_sigmoids(experts, top_k, device):
    """Whole logits from 38 on, whose sigmoid is 1 in 64 bits, with some far below."""
    rng = np.random.default_rng(experts + top_k)
    logits = rng.integers(38, rng.integers(40, 60, (500, 1)), (500, experts)).astype(np.float32)
    logits[rng.random(logits.shape) < rng.random((500, 1)) * 0.9] = -3.0
    logits += np.where(logits < 0, rng.integers(0, 9, logits.shape), 0).astype(np.float32)
    _, c = vc.route(vc.Tensor(logits, device=device), top_k, score="sigmoid")
    np.testing.assert_array_equal(c.numpy(), first_best(np.where(logits > 30, 100, logits), top_k))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [7, 30, 256, 300])
def test_logits_next_to_zero(experts, score, device):
    """Multiples of 2^-70, whose exponentials are 1 in 64 bits, with some of a tenth and more."""
    rng = np.random.default_rng(experts)
    logits = np.ldexp(rng.integers(-3, 4, (500, experts)), -70).astype(np.float32)
    far = rng.random(logits.shape) < 0.2
    logits[far] = (0.1 * rng.integers(-3, 4, far.sum())).astype(np.float32)
    for top_k in (1, 3):
        _, c = vc.route(vc.Tensor(logits, device=device), top_k, score=score)
        np.testing.assert_array_equal(c.numpy(), first_best(np.where(np.abs(logits) < 1e-3, 0, logits), top_k))
