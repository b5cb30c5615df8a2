"""The loss of a linear layer where the rows of its operands hold values unlike each other by many powers of two: features of raw
size, tokens and classes far from the others, and values in places that have no share in the result. Errors are held to float32's
roundings of the sums' own terms."""

import numpy as np
import pytest

import vectorcore_amd as vc
from test_linear_cross_entropy import DEVICES, UNIT, close, exact, problem, run

SIZES = [(9, 20, 30), (300, 64, 3000), (1100, 300, 9000)]
# Sizes whose products are packed: on either side of whole tiles and lines, sums that are split, rows in more than one piece.
PACKED = [(1000, 96, 3001), (256, 1024, 1024), (999, 515, 10007), (2049, 1030, 1537), (513, 1030, 6007), (257, 2050, 8200),
          (2000, 34, 9000), (70000, 64, 515)]
CASES = [(*s, "cpu") for s in SIZES[:2]] + [pytest.param(*s, "hip", marks=pytest.mark.gpu) for s in SIZES + PACKED]


def raw(rows, width, classes, size, seed=0):
    """One feature that is `size` times the others, say a date in seconds, with weights that make up for it."""
    x, w, t, b = problem(rows, width, classes, seed=seed)
    rng = np.random.default_rng(seed + rows)
    x[:, width // 3] = size * (1 + 0.25 * rng.random(rows))
    w[width // 3] /= np.float32(size)
    return x, w, t, b


def check(x, w, t, b, device, reduction="none", dy=None, keep=None):
    rows = len(x)
    dy = np.random.default_rng(rows).random(rows).astype(np.float32) if dy is None else dy
    loss, dx, dw, db = run(x, w, t, b, device, reduction, dy)
    number = max(1, (t >= 0).sum())
    share = dy.astype(np.float64) if reduction == "none" else 1 / number
    keep = np.arange(w.shape[1]) if keep is None else keep
    want, off = exact(x, w[:, keep], np.where(t >= 0, np.searchsorted(keep, t), -1), b[keep], share)
    if reduction == "none":
        close(loss, want["loss"], off["loss"])
    else:
        close(loss, want["loss"].sum() / number, off["loss"].sum() / number + 4 * UNIT * want["loss"].sum() / number)
    close(dx, want["dx"], off["dx"])
    close(dw[:, keep], want["dw"], off["dw"])
    close(db[keep], want["db"], off["db"])
    return loss, dx, dw, db


@pytest.mark.parametrize("size", [1e4, 1e6, 1.7e9, 1e12, 1e15])
@pytest.mark.parametrize("rows,width,classes,device", CASES[:2] + [pytest.param(1100, 300, 9000, "hip", marks=pytest.mark.gpu)])
def test_a_feature_of_raw_size(rows, width, classes, size, device):
    check(*raw(rows, width, classes, size), device)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,width,classes,device", CASES)
def test_a_feature_of_raw_size_in_calls_of_any_size(rows, width, classes, reduction, device):
    check(*raw(rows, width, classes, 1.7e9, seed=1), device, reduction)


@pytest.mark.parametrize("rows,width,classes,device", CASES)
def test_scores_with_a_feature_of_raw_size(rows, width, classes, device):
    x, w, t, b = raw(rows, width, classes, 1.7e9, seed=2)
    want, off = exact(x, w, t, b, 1.0)
    each = vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w)), t, bias=vc.Tensor(b, device=device), reduction="none")
    close(each.numpy(), want["loss"], off["loss"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_one_token_far_from_the_others(rows, width, classes, device):
    x, w, t, b = problem(rows, width, classes, seed=3, left_out=0)
    x[5, 3] = 3e11
    check(x, w, t, b, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_tokens_without_a_share_may_be_of_any_size(rows, width, classes, device):
    """Upstream gradients of zero for rows of 1e15, whose losses are of that size."""
    x, w, t, b = problem(rows, width, classes, seed=4)
    dy = np.random.default_rng(rows).random(rows).astype(np.float32)
    dy[::2] = 0
    x[::2] *= np.float32(1e15)
    check(x, w, t, b, device, dy=dy)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("every", [2, 3, 50])
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_classes_of_very_different_size(rows, width, classes, every, device):
    """Weights of some classes a trillionth of the others': their gradients and their rows' are as exact as the others'."""
    x, w, t, b = problem(rows, width, classes, seed=5)
    w[:, ::every] *= np.float32(1e-12)
    b[::every] += 3
    t = np.where(t >= 0, t // every * every, t)
    check(x, w, t, b, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mask", [-1e9, -1e30, np.finfo(np.float32).min])
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_masked_by_a_weight(rows, width, classes, mask, device):
    """A constant feature whose weights take every third class out."""
    x, w, t, b = problem(rows, width, classes, seed=6)
    x[:, 2] = 1
    out = np.arange(0, classes, 3)
    w[2, out] = mask
    t = np.where(t % 3 == 0, t + 1 - classes * (t + 1 >= classes) + (t + 1 >= classes), t)
    _, _, dw, db = check(x, w, t, b, device, keep=np.setdiff1d(np.arange(classes), out))
    assert (dw[:, out] == 0).all() and (db[out] == 0).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_rows_of_few_values(rows, width, classes, device):
    """Rows of one feature, of half of them, of none, and features that no row has."""
    x, w, t, b = problem(rows, width, classes, seed=7)
    x[np.random.default_rng(rows).random(x.shape) < 0.5] = 0
    x[::4] = 0
    x[np.arange(0, rows, 8), np.arange(0, rows, 8) % width] = 1
    x[:, -2] = 0
    w[5] = 0
    check(x, w, t, b, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_repeats_are_equal(rows, width, classes, device):
    x, w, t, b = raw(rows, width, classes, 1e9)
    runs = [run(x, w, t, b, device) for _ in range(3)]
    for again in runs[1:]:
        for a, c in zip(runs[0], again):
            np.testing.assert_array_equal(a, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 60])
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_upstream_gradients_of_any_size(rows, width, classes, scale, device):
    x, w, t, b = raw(rows, width, classes, 1e9)
    dy = (scale * np.random.default_rng(rows).random(rows)).astype(np.float32)
    check(x, w, t, b, device, dy=dy)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES + [(513, 1030, 6007)])
def test_a_weight_of_minus_infinity(rows, width, classes, device):
    """A constant feature whose weights of minus infinity take every third class out. That feature's own gradient is a sum of
    zeros times infinities, NaN; everything else is as without those classes."""
    if device == "cpu" and rows > 1000:
        rows, width, classes = 40, 100, 700
    x, w, t, b = problem(rows, width, classes, seed=8)
    x[:, 2] = 0.5
    out = np.arange(0, classes, 3)
    w[2, out] = -np.inf
    t = np.where(t % 3 == 0, 1, t)
    keep = np.setdiff1d(np.arange(classes), out)
    want, off = exact(x, w[:, keep], np.where(t >= 0, np.searchsorted(keep, t), -1), b[keep], 1.0)
    each = vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w)), t, bias=vc.Tensor(b, device=device), reduction="none")
    close(each.numpy(), want["loss"], off["loss"])
    loss, dx, dw, db = run(x, w, t, b, device, "none", np.ones(rows, np.float32))
    close(loss, want["loss"], off["loss"])
    counts = t >= 0
    others = np.delete(np.arange(width), 2)
    assert np.isnan(dx[counts, 2]).all() and (dx[~counts][:, others] == 0).all()
    close(dx[:, others], want["dx"][:, others], off["dx"][:, others])
    close(dw[:, keep], want["dw"], off["dw"])
    close(db[keep], want["db"], off["db"])
    assert (dw[:, out] == 0).all() and (db[out] == 0).all()
    t[0] = 0  # a class without a chance
    each = vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w)), t, bias=vc.Tensor(b, device=device),
                                   reduction="none").numpy()
    assert np.isposinf(each[0]) and np.isfinite(each[1:]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_infinite_logits_are_nan_in_their_rows_alone(rows, width, classes, device):
    """A logit of plus infinity has no loss; a row's infinity is its own."""
    x, w, t, b = problem(rows, width, classes, seed=9, left_out=0)
    scores = lambda x, w: vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w)), t, reduction="none").numpy()
    clean = exact(x, w, t, None, 1.0)
    dirty = x.copy()
    dirty[1, 4], dirty[3, 0] = np.inf, -np.inf
    each = scores(dirty, w)
    assert np.isnan(each[[1, 3]]).all()
    close(np.delete(each, [1, 3]), np.delete(clean[0]["loss"], [1, 3]), np.delete(clean[1]["loss"], [1, 3]))
    above = x[:, 6] > 0
    w[6, 3] = np.inf
    t[t == 3] = 4
    each, keep = scores(x, w), np.delete(np.arange(classes), 3)
    want, off = exact(x, w[:, keep], np.searchsorted(keep, t), None, 1.0)
    assert np.isnan(each[above]).all()  # plus infinity; minus infinity below zero
    close(each[~above], want["loss"][~above], off["loss"][~above])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,classes", SIZES)
def test_left_out_rows_beside_an_infinite_weight(rows, width, classes, device):
    """Their gradient is zero but for the feature of that weight, where it may be zero times infinity."""
    x, w, t, b = problem(rows, width, classes, seed=10, left_out=0.5)
    w[3, 5], t[0] = -np.inf, -1
    _, dx, _, _ = run(x, w, t, b, device, "none", np.ones(rows, np.float32))
    assert (np.delete(dx[t < 0], 3, 1) == 0).all()
