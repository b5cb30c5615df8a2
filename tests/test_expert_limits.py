"""The expert and router entry points at the ends of their ranges: no tokens."""

import ctypes

import numpy as np
import pytest

import vectorcore_amd as vc
from vectorcore_amd import cabi as C

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_of_no_tokens(device):
    z = lambda *s: vc.Tensor.zeros(s, device=device)
    x, gate, up, down = z(0, 5), z(3, 5, 7), z(3, 5, 7), z(3, 7, 4)
    for t in (x, gate, up, down):
        t.requires_grad = True
    plan = vc.ExpertPlan(z(0, 2), 3)
    rows = vc.expert_linear(vc.expert_gated(x, gate, up, plan), down, plan, ordered=True)
    y = vc.expert_combine(rows, z(0, 2), plan)
    assert tuple(y.shape) == (0, 4)
    y.backward(z(0, 4))
    assert tuple(x.grad.shape) == (0, 5)
    for t in (gate, up, down):
        np.testing.assert_array_equal(t.grad.numpy(), np.zeros(t.shape))


@pytest.mark.gpu
def test_a_plan_of_no_tokens_needs_no_words():
    lib = C.lib()
    plan = C.ExpertPlan(None, 0, 2, 3)
    out, out2 = C.Buffer.of(np.full(3 * 5 * 7, 9.0)), C.Buffer.of(np.full(3 * 5 * 7, 9.0))
    C.check(lib.vc_hip_expert_linear_backward_weight(None, None, out2.ptr, ctypes.byref(plan), 5, 7, 0, out.ptr, out2.ptr))
    assert (out.numpy() == 0).all() and (out2.numpy() == 0).all()
