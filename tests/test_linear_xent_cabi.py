"""The C entry points of the loss of a linear layer: the rows' losses and their mean of one call, on every route, and workspaces."""

import numpy as np
import pytest

from test_linear_cross_entropy import UNIT, close, exact, problem
from vectorcore_amd import cabi as C

pytestmark = pytest.mark.gpu


def forward(x, w, t, b, losses=True, mean=True):
    """What the call writes; buffers that it is not given keep the value they were filled with."""
    rows, width = x.shape
    held = [C.Buffer.of(v.astype(np.float32)) for v in (x, w, t)] + ([C.Buffer.of(b)] if b is not None else [])
    each, one = C.Buffer.of(np.full(rows, -7, np.float32)), C.Buffer.of(np.full(1, -7, np.float32))
    C.check(C.lib().vc_hip_linear_xent_forward(held[0].ptr, held[1].ptr, held[3].ptr if b is not None else None, held[2].ptr, rows,
                                               width, w.shape[1], each.ptr if losses else None, one.ptr if mean else None))
    return each.numpy(), one.numpy()[0]


# A few rows; float32 products in one piece, counted by each workgroup or before; in two pieces; packed products.
@pytest.mark.parametrize("rows,width,classes", [(5, 30, 700), (60, 40, 50), (1500, 20, 30), (33, 2, 2 ** 21), (1100, 300, 9000)])
def test_losses_and_mean_of_one_call(rows, width, classes):
    x, w, t, b = problem(rows, width, classes)
    want, off = exact(x, w, t, b, 1.0)
    number = (t >= 0).sum()
    each, mean = forward(x, w, t, b)
    close(each, want["loss"], off["loss"])
    close(mean, want["loss"].sum() / number, off["loss"].sum() / number + 4 * UNIT * want["loss"].sum() / number)
    alone, untouched = forward(x, w, t, b, mean=False)
    np.testing.assert_array_equal(alone, each)
    assert untouched == -7
    untouched, again = forward(x, w, t, b, losses=False)
    assert again == mean and (untouched == -7).all()


def workspace(rows, width, classes, step):
    """Bytes that a call with gradients of the weight and the bias takes from the pool."""
    lib = C.lib()
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((step, width))).astype(np.float32)
    w = (rng.standard_normal((width, classes)) / np.sqrt(width)).astype(np.float32)
    t = rng.integers(0, classes, rows).astype(np.float32)
    held = [C.Buffer.of(np.tile(x, (rows // step, 1))), C.Buffer.of(w), C.Buffer.of(t)]
    dw, db = C.Buffer((width, classes)), C.Buffer((classes,))
    C.synchronize()
    C.check(lib.vc_hip_pool_trim())
    before = C.pool_stats()
    C.check(lib.vc_hip_linear_xent_gradient(held[0].ptr, held[1].ptr, None, held[2].ptr, None, rows, width, classes, None, None, dw.ptr,
                                            db.ptr))
    C.synchronize()
    after = C.pool_stats()
    assert after.live_bytes == before.live_bytes
    got = db.numpy()
    # Of every class the probabilities' sum less its rows: zero together; each of `step` different rows often.
    z = x.astype(np.float64) @ w
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = p.mean(0) - np.bincount(t.astype(int), minlength=classes) / rows
    assert np.abs(got - want).max() <= 64 * UNIT * p.mean(0).max() + UNIT * 8 / rows
    return after.pooled_bytes


def test_workspace_of_many_pieces():
    """What does not hold a piece is a few numbers of each row. (A row of the bias's sums for every 256 rows of the call would
    be 240 bytes of each of these rows.)"""
    width, classes = 32, 7700
    few, many = (workspace(n * 65536, width, classes, 1024) for n in (4, 12))
    assert many - few <= 32 * 8 * 65536 + (64 << 20)
    # Logits and two packed copies of their gradients, of which this call needs one; less than a GiB for all else.
    assert many <= (2 << 30) + (3 << 30) + (1 << 30)
