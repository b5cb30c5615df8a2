"""Orthogonalised momentum updates against float64: the iterate itself, whole steps, batches of matrices, extreme
gradients, in-place semantics, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
A, B, C = 3.4445, -4.7750, 2.0315
UNIT = 2.0 ** -24


def exact(g, steps):
    x = g.astype(np.float64)
    norm = np.sqrt((x * x).sum((-2, -1), keepdims=True))
    x = np.divide(x, norm, out=np.zeros_like(x), where=norm != 0)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            gram = x @ np.swapaxes(x, -1, -2)
            x = A * x + (B * gram + C * gram @ gram) @ x
        else:
            gram = np.swapaxes(x, -1, -2) @ x
            x = A * x + x @ (B * gram + C * gram @ gram)
    return x


def near(shape, steps):
    """The iterate's error in the Frobenius norm. A step adds roundings that grow like the root of the terms added up, in
    three products whose factors' norms stay below 1.3 (30 = a + 2 |b| 1.3^2 + 3 |c| 1.3^4, rounded up), and passes earlier
    errors on at most 3.9-fold, the quintic's steepest slope on its range."""
    rows, cols = shape[-2:]
    step = 30 * np.sqrt(max(rows, cols) + 8) * UNIT * np.sqrt(min(rows, cols))
    return sum(step * 3.9 ** i for i in range(steps)) + 4 * UNIT


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 2), (3, 50), (50, 3), (31, 33), (64, 64), (65, 130), (200, 129), (10, 256), (256, 10),
          (128, 384), (5, 40, 24), (3, 24, 40), (2, 3, 17, 19), (140, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("steps", [0, 1, 5])
@pytest.mark.parametrize("shape", SHAPES)
def test_iterate(shape, steps, device):
    g = (1e-3 * np.random.default_rng(sum(shape)).standard_normal(shape)).astype(np.float32)
    o = vc.orthogonalise(vc.Tensor(g, device=device), steps=steps).numpy().astype(np.float64)
    error = np.sqrt(((o - exact(g, steps)) ** 2).sum((-2, -1)))
    assert (error <= near(shape, steps)).all()
    if steps == 5:
        values = np.linalg.svd(exact(g, 30), compute_uv=False)  # the definition's own range, reached early
        assert (np.linalg.svd(o, compute_uv=False).max(-1) <= max(values.max(), 1.3) + near(shape, steps)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 5, 65])
@pytest.mark.parametrize("shape", [(64, 256), (256, 64), (64, 257), (65, 256), (32, 512), (513, 32), (500, 9), (255, 33), (33, 33), (32, 1), (300, 7, 5),
                                   (3, 2, 61, 250)])
def test_iterate_around_the_largest_small_one(shape, steps):
    g = (1e-3 * np.random.default_rng(sum(shape)).standard_normal(shape)).astype(np.float32)
    o = vc.orthogonalise(vc.Tensor(g, device="hip"), steps=steps).numpy().astype(np.float64)
    if steps > 5:  # errors of singular values no longer shrink: their range alone is checked
        assert np.isfinite(o).all() and np.linalg.svd(o, compute_uv=False).max() < 1.3
        return
    error = np.sqrt(((o - exact(g, steps)) ** 2).sum((-2, -1)))
    assert (error <= near(shape, steps)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(60, 500, 630), (60, 630, 500), (33, 513, 769)])
def test_iterate_whose_last_round_of_tiles_is_split(count, rows, cols):
    """More tiles than the chip holds at once; the ones left over belong to several matrices."""
    g = (1e-3 * np.random.default_rng(count).standard_normal((count, rows, cols))).astype(np.float32)
    for steps in (1, 2):
        o = vc.orthogonalise(vc.Tensor(g, device="hip"), steps=steps).numpy().astype(np.float64)
        assert (np.sqrt(((o - exact(g, steps)) ** 2).sum((-2, -1))) <= near((rows, cols), steps)).all()


@pytest.mark.gpu
def test_steps_of_small_matrices_with_and_without_a_large_one():
    rng = np.random.default_rng(3)
    shapes = [(64, 256), (10, 7), (4, 30, 64), (200, 40), (1, 1), (256, 10)]

    def step(extra):
        def tensors(scale):
            return [vc.Tensor((scale * rng.standard_normal(s)).astype(np.float32), device="hip") for s in shapes]
        p, m, g = tensors(0.1), tensors(1e-3), tensors(1e-3)
        before = [[t.numpy() for t in ts] for ts in (p, m, g)]
        big = [vc.Tensor.zeros((300, 300), device="hip") for _ in range(3)] if extra else None
        vc.muon_step(p + big[:1] if extra else p, m + big[1:2] if extra else m, 0.02, momentum=0.9, weight_decay=0.1,
                     grads=g + big[2:] if extra else g)
        for shape, p0, m0, g0, p1, m1 in zip(shapes, *before, p, m):
            m_want = m0 * np.float32(0.9) + g0
            np.testing.assert_array_equal(m1.numpy(), m_want)
            rate = 0.02 * max(1.0, shape[-1] / shape[-2]) ** 0.5
            want = (1 - 0.02 * 0.1) * p0.astype(np.float64) - rate * exact(g0 + 0.9 * m_want.astype(np.float64), 5)
            # The iterate's input is off by a few roundings of its largest terms, which each step passes on 3.9-fold.
            error = np.sqrt(((p1.numpy() - want) ** 2).sum((-2, -1)))
            assert (error <= rate * (near(shape, 5) + 8 * UNIT * 3.9 ** 5) + 4 * UNIT * np.abs(p0).max() * np.sqrt(p0[..., 0].size + 1) * 16).all()

    step(False)
    step(True)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(700, 1500), (1501, 699), (24, 130, 258), (1100, 1100), (2, 300, 4097)])
def test_iterate_of_many_tiles(shape):
    g = (1e-3 * np.random.default_rng(sum(shape)).standard_normal(shape)).astype(np.float32)
    for steps in (1, 5):
        o = vc.orthogonalise(vc.Tensor(g, device="hip"), steps=steps).numpy().astype(np.float64)
        error = np.sqrt(((o - exact(g, steps)) ** 2).sum((-2, -1)))
        assert (error <= near(shape, steps)).all()


@pytest.mark.gpu
def test_more_parameters_than_a_launch_holds():
    rng = np.random.default_rng(5)
    shapes = [(int(a), int(b)) for a, b in rng.integers(1, 90, (31, 2))] + [(0, 7), (200, 300)]
    g = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    p = [vc.Tensor.zeros(s, device="hip") for s in shapes]
    m = [vc.Tensor.zeros(s, device="hip") for s in shapes]
    vc.muon_step(p, m, 1.0, momentum=0.0, grads=[vc.Tensor(a, device="hip") for a in g])
    for a, t, s in zip(g, p, shapes):
        if a.size:
            scale = np.sqrt(max(1.0, s[1] / s[0]))
            assert np.sqrt(((t.numpy() + scale * exact(a, 5)) ** 2).sum()) <= scale * (near(s, 5) + 8 * UNIT * np.sqrt(min(s)))


@pytest.mark.parametrize("device", DEVICES)
def test_extreme_matrices(device):
    rng = np.random.default_rng(3)
    u = rng.standard_normal((6, 20, 30)).astype(np.float32)
    u[0] = 0.0
    u[1] *= 1e30
    u[2] *= 1e-30
    u[3] = np.outer(u[3, :, 0], u[3, 0])       # rank one
    u[4] = 0.0
    u[4, 7, 9] = -1e-42                        # one denormal element
    u[5, 1:] *= 1e-20                          # one row beside nothing
    got = vc.orthogonalise(vc.Tensor(u, device=device)).numpy()
    assert (got[0] == 0).all()
    want = exact(u, 5)
    # Rows 1e-20 of the largest: an error relative to the norm, as everywhere.
    error = np.sqrt(((got - want) ** 2).sum((-2, -1)))
    assert (error <= near((20, 30), 5)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_not_a_number_stays_in_its_matrix(device):
    u = np.random.default_rng(4).standard_normal((3, 12, 8)).astype(np.float32)
    u[1, 2, 3] = np.nan
    got = vc.orthogonalise(vc.Tensor(u, device=device)).numpy()
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("given", [False, True])
def test_steps_of_several_parameters(given, device):
    rng = np.random.default_rng(12)
    shapes = [(40, 70), (70, 40), (33, 33), (4, 16, 24), (1, 5), (130, 260)]
    lr, mu, wd = 0.02, 0.9, 0.1
    p = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    m = [0.1 * rng.standard_normal(s).astype(np.float32) for s in shapes]
    m = [a.astype(np.float32) for a in m]
    tp = [vc.Tensor(a, requires_grad=True, device=device) for a in p]
    tm = [vc.Tensor(a, device=device) for a in m]
    p, m = [a.astype(np.float64) for a in p], [a.astype(np.float64) for a in m]
    for _ in range(3):
        g = [rng.standard_normal(s).astype(np.float32) for s in shapes]
        tg = [vc.Tensor(a, device=device) for a in g]
        versions = [t._version for t in tp + tm]
        if given:
            vc.muon_step(tp, tm, lr, momentum=mu, weight_decay=wd, grads=tg)
        else:
            vc.zero_grad(tp)
            for t, a in zip(tp, tg):
                (t * a).sum().backward()
            vc.muon_step(tp, tm, lr, momentum=mu, weight_decay=wd)
        assert all(t._version > v for t, v in zip(tp + tm, versions))
        for i, s in enumerate(shapes):
            m[i] = mu * m[i] + g[i]
            o = exact((g[i] + mu * m[i]).astype(np.float64), 5)
            p[i] = (1 - lr * wd) * p[i] - lr * np.sqrt(max(1.0, s[-1] / s[-2])) * o
    for i, s in enumerate(shapes):
        assert (np.abs(tm[i].numpy() - m[i]) <= 16 * UNIT * (np.abs(m[i]) + 4)).all()
        # The three updates' errors, and roundings of the parameter and of the update's direction (momenta a rounding
        # apart, passed on as an error of the normalised start).
        scale = lr * np.sqrt(max(1.0, s[-1] / s[-2]))
        error = np.sqrt(((tp[i].numpy() - p[i]) ** 2).sum((-2, -1)))
        limit = 3 * scale * (near(s, 5) + 3.9 ** 5 * 32 * UNIT * np.sqrt(min(s[-2:]))) + 16 * UNIT * np.sqrt((p[i] ** 2).sum((-2, -1)))
        assert (error <= limit).all()


@pytest.mark.parametrize("device", DEVICES)
def test_a_parameter_without_gradient_is_left_out(device):
    a, b = (vc.Tensor(np.ones((3, 4), np.float32), requires_grad=True, device=device) for _ in range(2))
    m = [vc.Tensor.zeros((3, 4), device=device) for _ in range(2)]
    (a * 2.0).sum().backward()
    vc.muon_step([a, b], m, 0.1)
    assert (b.numpy() == 1).all() and (m[1].numpy() == 0).all() and (m[0].numpy() == 2).all()
    assert (a.numpy() != 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_pending_reads_see_the_old_parameter(device):
    """A result that reads the parameter, taken before the step and read after it."""
    rng = np.random.default_rng(1)
    w, x, g = (rng.standard_normal((24, 24)).astype(np.float32) for _ in range(3))
    p = vc.Tensor(w, requires_grad=True, device=device)
    product, total = vc.Tensor(x, device=device) @ p, p + vc.Tensor(x, device=device)
    vc.muon_step([p], [vc.Tensor.zeros((24, 24), device=device)], 0.1, grads=[vc.Tensor(g, device=device)])
    np.testing.assert_allclose(product.numpy(), x.astype(np.float64) @ w, rtol=0, atol=32 * UNIT * (np.abs(x) @ np.abs(w)).max())
    np.testing.assert_array_equal(total.numpy(), x + w)
    assert (p.numpy() != w).any()
    with pytest.raises(RuntimeError, match="modified in place"):
        product.sum().backward() if product.requires_grad else None


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z = lambda *s: vc.Tensor.zeros(s, device=device)
    with pytest.raises(ValueError):
        vc.orthogonalise(z(4))
    p, m, g = z(3, 4), z(3, 4), z(3, 4)
    for args, kwargs in ((([p], []), dict(grads=[g])), (([p], [m]), dict(grads=[])), (([p], [z(4, 3)]), dict(grads=[g])),
                         (([p], [m]), dict(grads=[z(4, 3)])), (([z(5)], [z(5)]), dict(grads=[z(5)])),
                         (([p], [p]), dict(grads=[g])), (([p, p.reshape([4, 3])], [m, z(4, 3)]), dict(grads=[g, z(4, 3)])),
                         (([p], [m]), dict(grads=[m])), (([p], [m]), dict(grads=[p]))):
        with pytest.raises(ValueError):
            vc.muon_step(*args, 0.1, **kwargs)
    with pytest.raises(ValueError):
        vc.muon_step([p], [m], 0.1, grads=[g], steps=0)
    assert (p.numpy() == 0).all() and (m.numpy() == 0).all()
    vc.muon_step([], [], 0.1, grads=[])


@pytest.mark.gpu
def test_refuses_another_device():
    with pytest.raises(ValueError, match="device"):
        vc.muon_step([vc.Tensor.zeros((3, 4), device="hip")], [vc.Tensor.zeros((3, 4))], 0.1,
                     grads=[vc.Tensor.zeros((3, 4), device="hip")])
