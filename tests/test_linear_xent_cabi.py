"""The C entry points of the loss of a linear layer: the rows' losses and their mean of one call, on every route."""

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
