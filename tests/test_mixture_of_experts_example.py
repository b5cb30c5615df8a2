"""The mixture-of-experts example: it learns, and both devices take the same first steps."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

spec = importlib.util.spec_from_file_location(
    "mixture_of_experts", Path(__file__).resolve().parents[1] / "examples" / "mixture_of_experts.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize("device", ["cpu", pytest.param("hip", marks=pytest.mark.gpu)])
def test_it_learns(device):
    losses, right = example.train(device, steps=40, n=512)
    assert np.isfinite(losses).all() and losses[-1] < 0.2 * losses[0] and right > 0.95


@pytest.mark.gpu
def test_both_devices_take_the_same_first_steps():
    a, b = (example.train(device, steps=3, n=256)[0] for device in ("cpu", "hip"))
    # Losses of order one after steps whose errors (a few 1e-6 of the update) pass through a few hundred terms.
    np.testing.assert_allclose(a, b, rtol=2e-3)
