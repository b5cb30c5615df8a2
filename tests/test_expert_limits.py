"""The expert and router entry points at the ends of their ranges: no tokens, and picks up to 2^31."""

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


def window(buffer, begin, end):
    """Elements [begin, end) of a buffer of four-byte elements."""
    out = np.empty(end - begin, buffer.dtype)
    C.check(C.lib().vc_hip_download(out.ctypes.data, buffer.ptr + 4 * begin, out.nbytes))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [1, 2])
def test_a_plan_of_nearly_2_31_picks(top_k):
    """26 GB: all picks are of expert 0 but some at the end, where the last chunk ends behind 2^31."""
    lib, experts, tokens = C.lib(), 2, (2 ** 31 - 1) // top_k
    rows, words = tokens * top_k, ctypes.c_size_t()
    C.check(lib.vc_hip_expert_plan_words(tokens, top_k, experts, ctypes.byref(words)))
    chosen, plan = C.Buffer((rows,)), C.Buffer((words.value,), np.int32)
    C.check(lib.vc_hip_fill(chosen.ptr, rows, 0.0))
    tail = np.tile(np.array([1, 0, -1, 1, 0], np.float32), 400)
    C.check(lib.vc_hip_upload(chosen.ptr + 4 * (rows - len(tail)), tail.ctypes.data, tail.nbytes))
    C.check(lib.vc_hip_expert_plan_build(chosen.ptr, tokens, top_k, experts, plan.ptr))
    dropped, ones = (tail < 0).sum(), (tail == 1).sum()
    first = rows - dropped - ones
    offsets, token, place = 0, experts + 2, experts + 2 + rows
    np.testing.assert_array_equal(window(plan, offsets, token), [0, first, rows - dropped, rows])
    # Expert 0's picks but the tail's lie in their own order.
    head = rows - len(tail)
    for at in [0, 511, *range(2 ** 24 - 700, head - 2000, 2 ** 27), head - 2000]:
        some = np.arange(at, at + 1500)
        np.testing.assert_array_equal(window(plan, place + at, place + at + 1500), some)
        np.testing.assert_array_equal(window(plan, token + at, token + at + 1500), some // top_k)
    group = np.where(tail < 0, experts, tail).astype(int)
    order = np.argsort(group, kind="stable")
    starts = np.array([head, first, rows - dropped])
    want = np.empty(len(tail), np.int64)
    for g in range(3):
        mine = np.flatnonzero(group == g)
        want[mine] = starts[g] + np.arange(len(mine))
    np.testing.assert_array_equal(window(plan, place + head, place + rows), want)
    np.testing.assert_array_equal(window(plan, token + head, token + rows), (head + order) // top_k)
    for b in (chosen, plan):
        b.release()


@pytest.mark.gpu
def test_a_plan_of_no_tokens_needs_no_words():
    lib = C.lib()
    plan = C.ExpertPlan(None, 0, 2, 3)
    out, out2 = C.Buffer.of(np.full(3 * 5 * 7, 9.0)), C.Buffer.of(np.full(3 * 5 * 7, 9.0))
    C.check(lib.vc_hip_expert_linear_backward_weight(None, None, out2.ptr, ctypes.byref(plan), 5, 7, 0, out.ptr, out2.ptr))
    assert (out.numpy() == 0).all() and (out2.numpy() == 0).all()
