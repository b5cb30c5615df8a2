"""Layer normalisation and dropout of more than 2^32 values: what lies behind the first 16 GiB."""

import ctypes

import numpy as np
import pytest

from test_dropout import philox
from test_layer_norm import check
from vectorcore_amd import cabi as C

pytestmark = pytest.mark.gpu


class Buffer:
    def __init__(self, count, value=None):
        self.p = ctypes.c_void_p()
        C.check(C.lib().vc_hip_alloc(4 * count, ctypes.byref(self.p)))
        if value is not None:
            C.check(C.lib().vc_hip_fill(self.p, count, value))

    def at(self, offset):
        return ctypes.c_void_p(self.p.value + 4 * offset)

    def put(self, offset, values):
        C.check(C.lib().vc_hip_upload(self.at(offset), values.ctypes.data_as(ctypes.c_void_p), values.nbytes))

    def get(self, offset, count):
        out = np.empty(count, np.float32)
        C.check(C.lib().vc_hip_download(out.ctypes.data_as(ctypes.c_void_p), self.at(offset), out.nbytes))
        return out

    def __enter__(self):
        return self

    def __exit__(self, *_):
        C.check(C.lib().vc_hip_release(self.p))
        C.check(C.lib().vc_hip_synchronize())


def test_dropout_past_two_to_the_32():
    count, seed, stream = 2 ** 32 + 4099, 77, 5
    with Buffer(count, 1.0) as x, Buffer(count) as y:
        C.check(C.lib().vc_hip_dropout(x.p, None, count, 0.25, seed, stream, y.p))
        for first in (0, 2 ** 31 - 8, 2 ** 32 - 8, count - 11):
            n = min(16, count - first)
            want = [np.float32(1 / 0.75) if philox(i // 4, stream, seed)[i % 4] >= 2 ** 30 else 0 for i in range(first, first + n)]
            np.testing.assert_array_equal(y.get(first, n), want)
    C.check(C.lib().vc_hip_pool_trim())


@pytest.mark.parametrize("width", [1000, 16384, 40000])
def test_layer_norm_past_two_to_the_32(width):
    rows = 2 ** 32 // width + 3
    rng = np.random.default_rng(width)
    lib = C.lib()
    x_row, dy_row, w, b = (rng.standard_normal(width).astype(np.float32) for _ in range(4))
    with Buffer(rows * width, 0.5) as x, Buffer(rows * width, 0.0) as dy, Buffer(rows * width) as y, Buffer(4 * rows) as stats, \
            Buffer(width) as weight, Buffer(width) as bias, Buffer(width) as dw, Buffer(width) as db:
        weight.put(0, w)
        bias.put(0, b)
        last = (rows - 1) * width
        x.put(last, x_row)
        dy.put(last, dy_row)
        C.check(lib.vc_hip_layer_norm_forward(x.p, weight.p, bias.p, rows, width, 1e-5, y.p, stats.p))
        y_row, before = y.get(last, width), y.get(last - width, width)
        C.check(lib.vc_hip_layer_norm_backward(dy.p, x.p, weight.p, stats.p, rows, width, y.p, dw.p, db.p))
        check(x_row[None], w, b, float(np.float32(1e-5)), dy_row[None], y_row[None], y.get(last, width)[None], dw.get(0, width),
              db.get(0, width))
        np.testing.assert_array_equal(before, b)  # a constant row
        np.testing.assert_array_equal(y.get(last - width, width), np.zeros(width, np.float32))
    C.check(C.lib().vc_hip_pool_trim())
