"""How exact the packed products of the loss of a linear layer are: two half-precision parts from one, values far below the
largest of their row, rare classes beside frequent ones, and shares of very different size."""

import numpy as np
import pytest

import vectorcore_amd as vc
from test_linear_cross_entropy import UNIT, exact, problem, run

pytestmark = pytest.mark.gpu


def relative(got, want):
    return np.linalg.norm(np.asarray(got, np.float64) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("rows,width,classes", [(999, 515, 10007), (2049, 1030, 1537)])
def test_two_parts(rows, width, classes, reduction):
    """A part has 11 bits: products of one part alone are off by 2^-12 of each value, those without the second parts' products
    likewise. Two are off by 2^-22, of which sums keep the square root's share: far below 2^-18 of a result, also of one that
    cancels to a sixteenth of its terms."""
    x, w, t, b = problem(rows, width, classes)
    dy = np.random.default_rng(1).random(rows).astype(np.float32)
    got = run(x, w, t, b, "hip", reduction, dy)
    want, _ = exact(x, w, t, b, dy.astype(np.float64) if reduction == "none" else 1 / (t >= 0).sum())
    loss = want["loss"] if reduction == "none" else want["loss"].sum() / (t >= 0).sum()
    for a, b_, name in zip(got, (loss, want["dx"], want["dw"], want["db"]), ("loss", "dx", "dw", "db")):
        assert relative(a, b_) < 2.0 ** -18, name


def test_a_feature_far_above_the_others():
    """One feature is 2^18 times the others and has no weight: the others are held to 2^-39 of it, 2^-21 of themselves, which
    needs the half-precision numbers below 2^-14. The logits' errors are at most 2^-38 of the largest times the weights' sum."""
    rows, width, classes = 1100, 300, 9000
    x, w, t, b = problem(rows, width, classes, left_out=0)
    x[:, 17], w[17] = 2.0 ** 18 * 3, 0
    each = vc.linear_cross_entropy(vc.Tensor(x, device="hip"), vc.Tensor(w, device="hip"), t, bias=vc.Tensor(b, device="hip"),
                                   reduction="none").numpy()
    want, off = exact(x, w, t, b, 1.0)
    held = 2.0 ** -38 * np.abs(x).max() * np.abs(w).sum(0).max()
    assert (np.abs(each - want["loss"]) <= off["loss"] + 2 * held).all()
    assert relative(each, want["loss"]) < 2.0 ** -19  # flushed parts would leave 2^-12 of a logit's terms


def test_rare_classes_have_gradients_of_their_own():
    """Classes of probability 1e-12 to 1e-3: each column of the weight's gradient to a few roundings of its own size."""
    rows, width, classes = 1100, 300, 9000
    x, w, t, b = problem(rows, width, classes, sure=0.0, left_out=0)
    b -= np.linspace(0, 22, classes).astype(np.float32)
    t = np.minimum(t, classes // 50)
    _, _, dw, db = run(x, w, t, b, "hip")
    want, off = exact(x, w, t, b, 1 / rows)
    error = np.linalg.norm(dw - want["dw"], axis=0) / np.linalg.norm(want["dw"], axis=0)
    assert error.max() < 2.0 ** -17
    assert (np.abs(db - want["db"]) <= off["db"]).all()


@pytest.mark.parametrize("scale", [2.0 ** -60, 1.0, 2.0 ** 60])
def test_shares_of_very_different_size(scale):
    """Upstream gradients from 2^-70 to 1 times a scale, in blocks: a class's sums change their unit from block to block."""
    rows, width, classes = 1500, 260, 9000
    x, w, t, b = problem(rows, width, classes)
    rng = np.random.default_rng(8)
    dy = (rng.random(rows) * 2.0 ** -(10.0 * (np.arange(rows) // 128 % 8)) * scale).astype(np.float32)
    dy[300:600] = 0
    _, dx, dw, db = run(x, w, t, b, "hip", "none", dy)
    want, off = exact(x, w, t, b, dy.astype(np.float64))
    assert relative(dw, want["dw"]) < 2.0 ** -18 and relative(db, want["db"]) < 2.0 ** -18
    assert (np.abs(dw - want["dw"]) <= off["dw"] + UNIT * scale * 2.0 ** -60).all()
    counted = (t >= 0) & (dy != 0)
    error, size = np.linalg.norm(dx - want["dx"], axis=1)[counted], np.linalg.norm(want["dx"], axis=1)[counted]
    # The least step of float32 is 2^-149, by half of which each of a row's values is off: at a share of 2^-130 that is 2^-14.
    assert (error < 2.0 ** -16 * size + np.sqrt(width) * 2.0 ** -149).all()
    assert (dx[~counted] == 0).all()
