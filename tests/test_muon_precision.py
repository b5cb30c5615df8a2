"""The iterate of an orthogonalised update at float32's precision: its error against float64 next to that of the same
iteration in float32, for spectra that are flat, random, decaying and dominated by a row or a direction. Values held in
one half-precision number each would not pass."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
A, B, C = 3.4445, -4.7750, 2.0315
UNIT = 2.0 ** -24


def iterate(g, steps, dtype, keep=lambda v: v):
    """keep: what becomes of a value that is stored."""
    x = g.astype(np.float64)
    x = keep((x / np.sqrt((x * x).sum())).astype(dtype))
    if g.shape[0] > g.shape[1]:
        x = x.T
    for _ in range(steps):
        gram = keep((x @ x.T).astype(dtype))
        poly = keep((dtype(B) * gram + dtype(C) * (gram @ gram)).astype(dtype))
        x = keep((dtype(A) * x + poly @ x).astype(dtype))
    return (x if g.shape[0] <= g.shape[1] else x.T).astype(np.float64)


def norm(x):
    return np.sqrt((x * x).sum())


def limit(g, steps, want):
    """Sixteen times the error of the same iteration in float32, and sixteen roundings of the result. A value in two
    half-precision parts is off by 2^-22 of itself at most (4 UNIT, float32's by one), the product left out of two parts'
    four is 2^-22 of the largest: 12 UNIT a term for 2 or 3 in float32, whose sums round as often."""
    return 16 * norm(iterate(g, steps, np.float32) - want) + 16 * UNIT * norm(want)


def matrix(kind, rows, cols, seed):
    rng = np.random.default_rng(seed)
    g = rng.standard_normal((rows, cols))
    if kind == "flat":      # singular values alike
        u, _, v = np.linalg.svd(g, full_matrices=False)
        g = u @ v
    elif kind == "decaying":
        u, _, v = np.linalg.svd(g, full_matrices=False)
        g = (u * 2.0 ** (-np.arange(min(rows, cols)) / 6)) @ v
    elif kind == "row":     # one row of each side has nearly all: G and P start near one
        g[rows // 3] *= 300.0
    elif kind == "direction":
        g += 40.0 * np.sign(rng.standard_normal((rows, 1))) * np.sign(rng.standard_normal((1, cols)))
    return (1e-3 * g).astype(np.float32)


KINDS = ["flat", "random", "decaying", "row", "direction"]
CASES = [(kind, *shape) for kind in KINDS for shape in [(60, 200), (200, 129), (128, 384), (520, 300), (700, 1500)]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind,rows,cols", CASES)
def test_error_is_that_of_float32(kind, rows, cols, device):
    g = matrix(kind, rows, cols, rows)
    for steps in (1, 2, 5):
        want = iterate(g, steps, np.float64)
        got = vc.orthogonalise(vc.Tensor(g, device=device), steps=steps).numpy()
        assert norm(got - want) <= limit(g, steps, want), steps


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("count,rows,cols", [(60, 500, 630), (24, 130, 258), (40, 64, 256)])
def test_error_of_many_matrices(count, rows, cols, kind):
    """Tiles whose sums are split, of several matrices; small matrices of one launch."""
    g = np.stack([matrix(kind, rows, cols, 100 + i) for i in range(3)])
    many = np.concatenate([g] * (count // 3))
    for steps in (1, 5):
        got = vc.orthogonalise(vc.Tensor(many, device="hip"), steps=steps).numpy()
        for i in range(3):
            want = iterate(g[i], steps, np.float64)
            most = limit(g[i], steps, want)
            assert all(norm(o - want) <= most for o in got[i::3])


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(16, 26, 3266), (31, 3266, 26), (8, 60, 1000), (8, 200, 300), (40, 12, 700), (4, 130, 900)])
def test_error_is_no_larger_than_float32s(count, rows, cols):
    """Random matrices with a short side have nearly equal singular values, which pass a rounding on together. Half as much
    again as the same iterations in float32 leaves room for the luck of single roundings."""
    g = [matrix("random", rows, cols, 50 + i) for i in range(count)]
    got = vc.orthogonalise(vc.Tensor(np.stack(g), device="hip")).numpy()
    want = [iterate(a, 5, np.float64) for a in g]
    mine = norm(np.array([norm(o - w) for o, w in zip(got, want)]))
    float32 = norm(np.array([norm(iterate(a, 5, np.float32) - w) for a, w in zip(g, want)]))
    assert mine <= 1.5 * float32


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_at_float32s_precision(device):
    """The parameter itself: keep * p - rate * O, its own rounding beside the iterate's error."""
    rng = np.random.default_rng(8)
    for kind in KINDS:
        g, p, m = matrix(kind, 160, 300, 5), rng.standard_normal((160, 300)).astype(np.float32), matrix("random", 160, 300, 6)
        tp, tm = vc.Tensor(p, device=device), vc.Tensor(m, device=device)
        vc.muon_step([tp], [tm], 0.02, momentum=0.9, weight_decay=0.1, grads=[vc.Tensor(g, device=device)])
        next_m = m * np.float32(0.9) + g
        np.testing.assert_array_equal(tm.numpy(), next_m)
        u = g + np.float32(0.9) * next_m
        want = iterate(u, 5, np.float64)
        rate = 0.02 * np.sqrt(300 / 160)
        error = norm(tp.numpy() - ((1 - 0.02 * 0.1) * p.astype(np.float64) - rate * want))
        assert error <= rate * limit(u, 5, want) + 4 * UNIT * norm(p.astype(np.float64))


@pytest.mark.parametrize("kind,rows,cols", CASES)
def test_one_half_each_would_not_pass(kind, rows, cols):
    """The bound tells two parts from one: values stored as their first parts alone exceed it everywhere."""
    g = matrix(kind, rows, cols, rows)
    half = lambda v: (v * np.float32(2.0 ** 14)).astype(np.float16).astype(np.float32) / np.float32(2.0 ** 14)
    for steps in (1, 5):
        want = iterate(g, steps, np.float64)
        assert norm(iterate(g, steps, np.float32, half) - want) > 4 * limit(g, steps, want)
