"""The router of a mixture of experts against its definition in float64: which experts are chosen and in which order
(ties, borders between ranks, groups, NaN and infinities), their weights, the gradient to the logits, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24


def exact(logits, top_k, bias=None, score="softmax", groups=1, top_groups=1, renormalise=True, grad=None):
    with np.errstate(all="ignore"):
        l = logits.astype(np.float64)
        if score == "sigmoid":
            s = 1 / (1 + np.exp(-l))
        else:
            s = np.exp(l - l.max(1, keepdims=True))
            s /= s.sum(1, keepdims=True)
        ranks = s if bias is None else s + bias.astype(np.float64)
        tokens, experts = l.shape
        first = np.where(np.isnan(ranks), np.inf, ranks)  # a NaN ranks first
        size = experts // groups
        if groups > 1:
            strength = np.sort(first.reshape(tokens, groups, size), 2)[:, :, -2:].sum(2)
            kept = np.argsort(-strength, axis=1, kind="stable")[:, :top_groups]
            is_open = np.zeros((tokens, groups), bool)
            np.put_along_axis(is_open, kept, True, 1)
            closed = ~np.repeat(is_open, size, axis=1)
        else:
            closed = np.zeros((tokens, experts), bool)
        order = np.lexsort((np.broadcast_to(np.arange(experts), (tokens, experts)), -first, closed), axis=1)
        chosen = order[:, :top_k]
        p = np.take_along_axis(s, chosen, 1)
        total = p.sum(1, keepdims=True) if renormalise else np.ones((tokens, 1))
        if grad is None:
            return p / total, chosen
        g = grad.astype(np.float64)
        dp = (g - (g * p).sum(1, keepdims=True) / total) / total if renormalise else g
        ds = np.zeros_like(s)
        np.put_along_axis(ds, chosen, dp, 1)
        d = ds * s * (1 - s) if score == "sigmoid" else s * (ds - (ds * s).sum(1, keepdims=True))
        return p / total, chosen, d


CASES = [(1, 1, 1, 1, 1), (3, 2, 2, 1, 1), (1, 64, 4, 8, 4), (65, 33, 5, 1, 1), (65, 33, 5, 3, 2), (7, 63, 8, 1, 1),
         (7, 65, 3, 5, 1), (130, 128, 8, 2, 1), (5, 129, 1, 1, 1), (66, 256, 8, 8, 4), (9, 257, 6, 1, 1), (3, 512, 8, 64, 9),
         (2, 1000, 64, 4, 3), (2, 1024, 33, 16, 5), (12, 48, 8, 48, 8), (0, 8, 2, 1, 1), (1027, 16, 2, 4, 4)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k,groups,top_groups", CASES)
def test_choice_weights_and_gradient(tokens, experts, top_k, groups, top_groups, renormalise, score, device):
    rng = np.random.default_rng(tokens + 31 * experts + top_k)
    logits = rng.standard_normal((tokens, experts)).astype(np.float32)
    bias = (0.02 * rng.standard_normal(experts)).astype(np.float32) if (experts + top_k) % 2 else None
    grad = rng.standard_normal((tokens, top_k)).astype(np.float32)
    l = vc.Tensor(logits, requires_grad=True, device=device)
    w, c = vc.route(l, top_k, bias=None if bias is None else vc.Tensor(bias, device=device), score=score, groups=groups,
                    top_groups=top_groups, renormalise=renormalise)
    assert not c.requires_grad and tuple(w.shape) == tuple(c.shape) == (tokens, top_k)
    w.backward(vc.Tensor(grad, device=device))
    want_w, want_c, want_d = exact(logits, top_k, bias, score, groups, top_groups, renormalise, grad)
    np.testing.assert_array_equal(c.numpy().reshape(tokens, top_k), want_c)
    # A score is an exponential (its argument off by a rounding of a number below 16), a sum and a quotient, each of a
    # few roundings; the sum adds at most log2 of the experts more.
    rel = (48 + 2 * np.log2(experts + 1)) * UNIT
    np.testing.assert_allclose(w.numpy().reshape(tokens, top_k), want_w, rtol=rel, atol=1e-38)
    # The gradient's terms: at most |g| times a score (over the chosen scores' sum), which may cancel.
    p = want_w if renormalise else want_w
    scale = (np.abs(grad).max(1, keepdims=True) + np.abs(grad * p).sum(1, keepdims=True)) if tokens else 0
    assert (np.abs(l.grad.numpy().reshape(tokens, experts) - want_d) <= 4 * rel * scale + 1e-37).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_equal_ranks_go_to_the_lower_index(score, groups, top_groups, device):
    rng = np.random.default_rng(7)
    logits = rng.integers(0, 3, (257, 64)).astype(np.float32)
    logits[0] = 1.5
    _, c = vc.route(vc.Tensor(logits, device=device), 8, score=score, groups=groups, top_groups=top_groups)
    np.testing.assert_array_equal(c.numpy(), exact(logits, 8, None, score, groups, top_groups)[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ranks_a_rounding_apart(score, with_bias, device):
    """Logits one float apart, in falling and rising order of their index: a choice by 32-bit scores would tie."""
    tokens, experts = 64, 96
    logits = np.full((tokens, experts), 0.25, np.float32)
    for e in range(1, experts):
        logits[:, e] = np.nextafter(logits[:, e - 1], np.float32(1))
    logits[::2] = logits[::2, ::-1]
    bias = np.full(experts, 0.125, np.float32) if with_bias else None
    for groups, top_groups in ((1, 1), (8, 3)):
        _, c = vc.route(vc.Tensor(logits, device=device), 6, score=score, groups=groups, top_groups=top_groups,
                        bias=vc.Tensor(bias, device=device) if with_bias else None)
        np.testing.assert_array_equal(c.numpy(), exact(logits, 6, bias, score, groups, top_groups)[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups", [(256, 8, 3), (256, 1, 1), (128, 16, 5), (64, 16, 9), (192, 3, 2), (96, 8, 4)])
@pytest.mark.parametrize("centre,spread", [(0.0, 1e-4), (-1.0, 1e-6), (3.0, 1e-7), (-30.0, 1.0), (-70.0, 4.0), (-90.0, 3.0)])
@pytest.mark.parametrize("bias_scale", [1e-5, 1.0, 300.0])
def test_ranks_at_all_distances(bias_scale, centre, spread, experts, groups, top_groups, score, device):
    """Distances from far below 32 bits' to far above them, of scores and biases alone and together."""
    rng = np.random.default_rng(experts + groups)
    steps = np.exp(rng.uniform(-6, 0, (65, experts))) * rng.choice([-1, 1], (65, experts))
    logits = (centre + spread * steps).astype(np.float32)
    bias = (bias_scale * rng.choice([-1.0, 0.5, 0.5, 0.5, 1.0], experts)).astype(np.float32)
    _, c = vc.route(vc.Tensor(logits, device=device), 7, score=score, groups=groups, top_groups=top_groups,
                    bias=vc.Tensor(bias, device=device))
    want = exact(logits, 7, bias, score, groups, top_groups)[1]
    # Where 64 bits, too, cannot tell two ranks or groups' sums apart, the choice is either's: those rows are left out.
    l = logits.astype(np.float64)
    s = 1 / (1 + np.exp(-l)) if score == "sigmoid" else np.exp(l - l.max(1, keepdims=True))
    ranks = (s if score == "sigmoid" else s / s.sum(1, keepdims=True)) + bias
    least = 64 * np.finfo(np.float64).eps * np.abs(ranks).max()
    strength = np.sort(np.sort(ranks.reshape(65, groups, -1), 2)[:, :, -2:].sum(2), 1)
    cut = strength[:, -top_groups] - strength[:, -top_groups - 1] if top_groups < groups else np.full(65, np.inf)
    kept = np.argsort(-np.sort(ranks.reshape(65, groups, -1), 2)[:, :, -2:].sum(2), axis=1, kind="stable")[:, :top_groups]
    is_open = (kept[:, :, None] == np.arange(experts) // (experts // groups)).any(1)
    best = np.sort(np.where(is_open, ranks, -np.inf), 1)[:, ::-1][:, :8]
    clear = (np.minimum(cut, (best[:, :-1] - best[:, 1:]).min(1)) > least)
    np.testing.assert_array_equal(c.numpy()[clear], want[clear])
    if centre == 0.0 and bias_scale < 1e-3:
        assert clear.sum() > 50


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_special_values(score, renormalise, device):
    """Masked experts (-inf), the lowest number, rows whose mask leaves nothing, NaN, +inf, saturated scores."""
    low = np.finfo(np.float32).min
    logits = np.random.default_rng(2).standard_normal((12, 24)).astype(np.float32)
    logits[0, :20] = -np.inf
    logits[1, :] = -np.inf
    logits[2, 5:] = low
    logits[3, :] = low
    logits[4, 7] = np.nan
    logits[5, 3] = np.inf
    logits[6, [3, 9]] = np.inf
    logits[7, 2], logits[7, 4] = np.nan, np.inf
    logits[8, 11] = 90.0
    logits[9, :] = np.finfo(np.float32).max
    logits[10] *= 30.0
    w, c = vc.route(vc.Tensor(logits, device=device), 3, score=score, renormalise=renormalise)
    want_w, want_c = exact(logits, 3, None, score, renormalise=renormalise)
    np.testing.assert_array_equal(c.numpy(), want_c)
    np.testing.assert_allclose(w.numpy(), want_w, rtol=256 * UNIT, atol=2e-38)


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    rng = np.random.default_rng(11)
    logits = rng.standard_normal((4, 12)).astype(np.float32)
    grad = rng.standard_normal((4, 3)).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            l = vc.Tensor(logits, requires_grad=True, device=device)
            w, c = vc.route(l, 3, score=score, renormalise=renormalise)
            w.backward(vc.Tensor(grad, device=device))
            got, at = l.grad.numpy(), c.numpy().astype(int)
            for t, e in ((0, at[0, 0]), (1, at[1, 2]), (2, (at[2, 0] + 1) % 12), (3, 5)):
                h, values = 1e-6, []
                for sign in (1, -1):
                    moved = logits.astype(np.float64)
                    moved[t, e] += sign * h
                    s = 1 / (1 + np.exp(-moved[t])) if score == "sigmoid" else np.exp(moved[t]) / np.exp(moved[t]).sum()
                    p = s[at[t]]
                    values.append((grad[t] * (p / p.sum() if renormalise else p)).sum())
                # A central difference's own error: its step squared, and a double's rounding over the step.
                assert abs(got[t, e] - (values[0] - values[1]) / (2 * h)) <= 1e-6


@pytest.mark.parametrize("device", DEVICES)
def test_saved_logits_are_checked(device):
    l = vc.Tensor(np.ones((3, 4), np.float32), requires_grad=True, device=device)
    w, _ = vc.route(l, 2)
    total = w.sum()
    total.backward()
    vc.sgd_step([l], 0.5)
    with pytest.raises(RuntimeError, match="modified in place"):
        total.backward()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    l = vc.Tensor(np.zeros((3, 12), np.float32), device=device)
    for kwargs in (dict(top_k=0), dict(top_k=13), dict(top_k=2, score="relu"), dict(top_k=2, groups=0),
                   dict(top_k=2, groups=5), dict(top_k=2, groups=4, top_groups=0), dict(top_k=2, groups=4, top_groups=5),
                   dict(top_k=4, groups=4, top_groups=1), dict(top_k=2, bias=vc.Tensor(np.zeros(11, np.float32), device=device))):
        with pytest.raises(ValueError):
            vc.route(l, **kwargs)
    for shape in ((12,), (2, 3, 12), (2, 0), (2, 1025)):
        with pytest.raises(ValueError):
            vc.route(vc.Tensor.zeros(shape, device=device), 1)
    with pytest.raises(ValueError):
        vc.route(vc.Tensor.zeros((2, 128), device=device), 65)


@pytest.mark.gpu
def test_refuses_a_bias_on_another_device():
    with pytest.raises(ValueError, match="device|is on"):
        vc.route(vc.Tensor.zeros((2, 8), device="hip"), 2, bias=vc.Tensor.zeros((8,), device="cpu"))
