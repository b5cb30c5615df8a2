"""The router where the chosen scores are far below one, or next to one: weights and gradients are ratios of scores and
distances from one, which stay ordinary numbers where the scores do not. Against float64, in logarithms."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


def exact(logits, chosen, score, renormalise, grad):
    """The weights of the given choice, the gradient to the logits, and the size of the terms that it adds up."""
    l = logits.astype(np.float64)
    if score == "sigmoid":
        logs = np.minimum(l, 0) - np.log1p(np.exp(-np.abs(l)))
    else:
        top = l.max(1, keepdims=True)
        logs = l - top - np.log(np.exp(l - top).sum(1, keepdims=True))
    picked = np.take_along_axis(logs, chosen, 1)
    w = np.exp(picked)
    if renormalise:
        w = np.exp(picked - picked.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
    g = grad.astype(np.float64)
    mean, size = (g * w).sum(1, keepdims=True), (np.abs(g) * w).sum(1, keepdims=True)
    d, scale = np.zeros_like(l), np.zeros_like(l)
    if score == "softmax" and not renormalise:
        np.put_along_axis(d, chosen, g, 1)
        return w, np.exp(logs) * (d - mean), np.exp(logs) * (np.abs(d) + size)
    outer = w
    if score == "sigmoid":
        x = np.take_along_axis(l, chosen, 1)
        outer = w * np.exp(np.minimum(-x, 0) - np.log1p(np.exp(-np.abs(x))))  # times what is missing to one
    np.put_along_axis(d, chosen, outer * (g - mean if renormalise else g), 1)
    np.put_along_axis(scale, chosen, outer * (np.abs(g) + (size if renormalise else 0)), 1)
    return w, d, scale


def check(logits, top_k, score, renormalise, device, **kwargs):
    rng = np.random.default_rng(top_k)
    grad = rng.standard_normal((len(logits), top_k)).astype(np.float32)
    l = vc.Tensor(logits, requires_grad=True, device=device)
    w, c = vc.route(l, top_k, score=score, renormalise=renormalise, **kwargs)
    w.backward(vc.Tensor(grad, device=device))
    chosen = c.numpy().astype(int)
    want_w, want_d, scale = exact(logits, chosen, score, renormalise, grad)
    # An exponential, its argument off by a rounding of a number below 16, a sum over the experts and a quotient. What
    # lies below the least normal number has fewer bits.
    rel = (48 + 2 * np.log2(logits.shape[1] + 1)) * UNIT
    np.testing.assert_allclose(w.numpy(), want_w, rtol=rel, atol=1e-38)
    assert (np.abs(l.grad.numpy() - want_d) <= 4 * rel * scale + 1e-37).all()
    return chosen


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("experts,top_k", [(16, 1), (16, 3), (200, 8), (300, 5)])
@pytest.mark.parametrize("centre", [-200.0, -120.0, -103.0, -96.0, -89.0, -80.0, 12.0, 30.0, 85.0, 95.0])
def test_sigmoid_scores(centre, experts, top_k, renormalise, device):
    rng = np.random.default_rng(experts)
    logits = (centre + rng.uniform(-7, 7, (65, experts))).astype(np.float32)
    chosen = check(logits, top_k, "sigmoid", renormalise, device)
    if centre < 0:
        np.testing.assert_array_equal(chosen, np.argsort(-logits, axis=1, kind="stable")[:, :top_k])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("depth", [70.0, 92.0, 100.0, 140.0])
@pytest.mark.parametrize("experts,groups", [(32, 1), (32, 4), (256, 8), (320, 1)])
def test_a_bias_prefers_small_scores(experts, groups, depth, score, renormalise, device):
    """One expert has nearly all of the softmax, and the bias keeps it from being chosen."""
    rng = np.random.default_rng(int(depth))
    logits = (-depth + rng.uniform(-7, 7, (65, experts))).astype(np.float32)
    logits[:, 0] = 3.0
    bias = (1.0 + rng.permutation(experts) / 16.0).astype(np.float32)
    bias[:experts // groups if groups > 1 else 1] = -10.0
    kwargs = dict(bias=vc.Tensor(bias, device=device), groups=groups, top_groups=max(1, groups // 2))
    chosen = check(logits, 6 if groups < 8 else 4, score, renormalise, device, **kwargs)
    assert (chosen > 0).all()
    if groups == 1:
        np.testing.assert_array_equal(chosen, np.broadcast_to(np.argsort(-bias, kind="stable")[:6], chosen.shape))


@pytest.mark.parametrize("device", DEVICES)
def test_two_small_scores(device):
    logits = np.full((3, 8), -200.0, np.float32)
    logits[:, 2:4] = [[-88.0, -89.0], [-90.0, -91.0], [-87.5, -120.0]]
    l = vc.Tensor(logits, requires_grad=True, device=device)
    w, c = vc.route(l, 2, score="sigmoid")
    np.testing.assert_array_equal(c.numpy(), [[2, 3]] * 3)
    np.testing.assert_allclose(w.numpy()[:2], [[0.7310585786, 0.2689414214]] * 2, rtol=64 * UNIT)
    w.backward(vc.Tensor(np.array([[1, -1], [1, 0], [0.5, 0.5]], np.float32), device=device))
    slope = 0.7310585786 * 0.2689414214
    np.testing.assert_allclose(l.grad.numpy()[:2, 2:4], [[2 * slope, -2 * slope], [slope, -slope]], rtol=64 * UNIT)
    np.testing.assert_allclose(l.grad.numpy()[2], np.zeros(8), atol=64 * UNIT)
