"""The expert and router entry points at the ends of their ranges: no tokens, picks up to 2^31, and more
workgroups than one dimension of a grid holds."""

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


def windows(buffer, width, rows):
    """Rows [begin, end) of a buffer at its start, inside and at its end."""
    for at in (0, rows // 2, 2 ** 26 - 700, rows - 1500):
        yield at, window(buffer, at * width, (at + 1500) * width).reshape(1500, width)


def filled(*shape, value=7.0):
    b = C.Buffer(shape)
    C.check(C.lib().vc_hip_fill(b.ptr, int(np.prod(shape, dtype=np.int64)), value))
    return b


@pytest.mark.gpu
def test_a_sum_over_more_than_2_26_picks():
    lib, tokens, width = C.lib(), 2 ** 25 + 1000, 3
    rows, words = 2 * tokens, ctypes.c_size_t()
    C.check(lib.vc_hip_expert_plan_words(tokens, 2, 1, ctypes.byref(words)))
    chosen, plan = filled(rows, value=0.0), C.Buffer((words.value,), np.int32)
    C.check(lib.vc_hip_expert_plan_build(chosen.ptr, tokens, 2, 1, plan.ptr))
    p = C.ExpertPlan(plan.ptr, tokens, 2, 1)
    z, w, g = filled(rows, width, value=3.0), filled(rows, value=0.5), filled(tokens, width, value=2.0)
    out, dz, dw = filled(tokens, width), filled(rows, width), filled(rows)
    C.check(lib.vc_hip_expert_combine_forward(z.ptr, w.ptr, ctypes.byref(p), width, out.ptr))
    C.check(lib.vc_hip_expert_combine_backward(g.ptr, z.ptr, w.ptr, ctypes.byref(p), width, dz.ptr, dw.ptr))
    assert (window(out, 3 * (tokens - 1500), 3 * tokens) == 3.0).all()
    assert all((v == 1.0).all() for _, v in windows(dz, width, rows))
    assert all((v == 18.0).all() for _, v in windows(dw, 1, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top_k", [(2 ** 28 + 999, 2, 1), (2 ** 26 + 999, 17, 17)])
def test_routes_of_more_rows_than_a_grids_dimension(tokens, experts, top_k):
    """All rows are alike but windows of them, whose second expert is the best."""
    lib = C.lib()
    logits, w, c = filled(tokens, experts, value=0.0), filled(tokens, top_k), filled(tokens, top_k)
    some = np.zeros((1500, experts), np.float32)
    some[:, 1] = 1.0
    for at, _ in windows(logits, experts, tokens):
        C.check(lib.vc_hip_upload(logits.ptr + 4 * at * experts, some.ctypes.data, some.nbytes))
    C.check(lib.vc_hip_route_forward(logits.ptr, None, tokens, experts, top_k, C.SOFTMAX, 1, 1, 0, w.ptr, c.ptr))
    order = [1, 0, *range(2, experts)][:top_k]
    p = np.exp(some[0].astype(np.float64)) / np.exp(some[0].astype(np.float64)).sum()
    for _, v in windows(c, top_k, tokens):
        np.testing.assert_array_equal(v, np.broadcast_to(order, v.shape))
    for _, v in windows(w, top_k, tokens):
        np.testing.assert_allclose(v, np.broadcast_to(p[order], v.shape), rtol=2.0 ** -19)
    if experts > 2:
        return
    g, d = filled(tokens, 1, value=1.0), filled(tokens, 2)
    C.check(lib.vc_hip_route_backward(logits.ptr, c.ptr, g.ptr, tokens, 2, 1, C.SOFTMAX, 0, d.ptr))
    for _, v in windows(d, 2, tokens):
        np.testing.assert_allclose(v, np.broadcast_to([-p[0] * p[1], p[0] * p[1]], v.shape), rtol=2.0 ** -18)


@pytest.mark.gpu
def test_too_many_tiles_are_refused():
    """2^24 workgroups of 256 and more; nothing is launched."""
    lib, p = C.lib(), C.Buffer((16,))
    plan = C.ExpertPlan(p.ptr, 1 << 20, 1, 8)
    most = 1 << 20
    for call in (lambda: lib.vc_hip_expert_linear_forward(p.ptr, p.ptr, ctypes.byref(plan), 4, most, 0, p.ptr),
                 lambda: lib.vc_hip_expert_gated_forward(p.ptr, p.ptr, p.ptr, ctypes.byref(plan), 4, most, 0, p.ptr, None, None),
                 lambda: lib.vc_hip_expert_linear_backward_input(p.ptr, p.ptr, None, None, ctypes.byref(plan), most, 4, p.ptr),
                 lambda: lib.vc_hip_expert_linear_backward_weight(p.ptr, p.ptr, None, ctypes.byref(plan), most, most, 0, p.ptr, None)):
        assert call() == 3 and b"too many tiles" in lib.vc_hip_last_error()


@pytest.mark.gpu
def test_a_plan_of_no_tokens_needs_no_words():
    lib = C.lib()
    plan = C.ExpertPlan(None, 0, 2, 3)
    out, out2 = C.Buffer.of(np.full(3 * 5 * 7, 9.0)), C.Buffer.of(np.full(3 * 5 * 7, 9.0))
    C.check(lib.vc_hip_expert_linear_backward_weight(None, None, out2.ptr, ctypes.byref(plan), 5, 7, 0, out.ptr, out2.ptr))
    assert (out.numpy() == 0).all() and (out2.numpy() == 0).all()
