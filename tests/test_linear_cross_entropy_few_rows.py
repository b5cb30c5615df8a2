"""Scores of up to seventeen rows on either side of the rule that reads the weight once for them: many classes and few, few
features and very many."""

import numpy as np
import pytest

import vectorcore_amd as vc
from test_linear_cross_entropy import DEVICES, UNIT, close, exact, problem


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17])
@pytest.mark.parametrize("width,classes", [(5, 16001), (130, 16127), (260, 50003), (515, 33000), (700, 129), (4100, 1000), (9000, 3)])
def test_scores(rows, width, classes):
    x, w, t, b = problem(rows, width, classes)
    t[0] = classes - 1
    want, off = exact(x, w, t, b, 1.0)
    each = vc.linear_cross_entropy(*(vc.Tensor(v, device="hip") for v in (x, w)), t, bias=vc.Tensor(b, device="hip"), reduction="none")
    close(each.numpy(), want["loss"], off["loss"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 7, 16])
def test_a_million_features(rows, device):
    """Terms of one sign and size, whose roundings do not cancel: a chain of n of them is off by up to n / 2 roundings of the
    whole; these are held to the 4 sqrt(n) of terms of any sign."""
    width = 2 ** 20 + 5
    x = np.full((rows, width), 1.0, np.float32) + np.arange(rows, dtype=np.float32)[:, None] / 64
    w = np.outer(np.ones(width), [1.1, 1.1001, 1.0999]).astype(np.float32) / np.float32(2 ** 17)
    t = np.arange(rows) % 3
    want, off = exact(x, w, t, None, 1.0)
    each = vc.linear_cross_entropy(*(vc.Tensor(v, device=device) for v in (x, w)), t, reduction="none")
    close(each.numpy(), want["loss"], off["loss"])
