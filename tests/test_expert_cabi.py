"""Refusals of the C entry points of the router, the experts and the orthogonalised update: a status and a message, nothing
launched."""

import ctypes

import pytest

from vectorcore_amd import cabi as C


def calls(lib, p):
    """(status code, call) pairs; p: a device pointer that no refused call reads."""
    plan = C.ExpertPlan(p, 4, 2, 8)
    none, many = C.ExpertPlan(None, 4, 2, 8), C.ExpertPlan(p, 4, 2, 2000)
    huge = C.ExpertPlan(p, 1 << 40, 2, 8)
    words = ctypes.c_size_t()
    item = lambda **kw: (C.MuonItem * 1)(C.MuonItem(**dict(dict(param=p, momentum=p, grad=p, count=1, rows=4, cols=4), **kw)))
    route = lambda **kw: (lambda a: lib.vc_hip_route_forward(a["logits"], None, 3, a["experts"], a["top_k"], a["score"], a["groups"],
                                                            a["top_groups"], 1, a["weights"], p))(
        dict(dict(logits=p, experts=8, top_k=2, score=0, groups=1, top_groups=1, weights=p), **kw))
    return [
        (1, lambda: route(experts=0)), (1, lambda: route(experts=1025)), (1, lambda: route(top_k=0)), (1, lambda: route(top_k=9)),
        (1, lambda: route(score=2)), (1, lambda: route(groups=3)), (1, lambda: route(groups=4, top_groups=5)),
        (1, lambda: route(groups=8, top_groups=1)), (1, lambda: route(logits=None)), (1, lambda: route(weights=None)),
        (1, lambda: lib.vc_hip_route_backward(p, p, None, 3, 8, 2, 0, 1, p)),
        (1, lambda: lib.vc_hip_route_backward(p, p, p, 3, 8, 9, 0, 1, p)),
        (1, lambda: lib.vc_hip_expert_plan_words(4, 0, 8, ctypes.byref(words))),
        (1, lambda: lib.vc_hip_expert_plan_words(4, 2, 0, ctypes.byref(words))),
        (3, lambda: lib.vc_hip_expert_plan_words(1 << 31, 2, 8, ctypes.byref(words))),
        (1, lambda: lib.vc_hip_expert_plan_build(None, 4, 2, 8, p)), (1, lambda: lib.vc_hip_expert_plan_build(p, 4, 2, 8, None)),
        (1, lambda: lib.vc_hip_expert_linear_forward(p, p, ctypes.byref(none), 4, 4, 0, p)),
        (1, lambda: lib.vc_hip_expert_linear_forward(p, p, None, 4, 4, 0, p)),
        (1, lambda: lib.vc_hip_expert_linear_forward(p, p, ctypes.byref(many), 4, 4, 0, p)),
        (3, lambda: lib.vc_hip_expert_linear_forward(p, p, ctypes.byref(huge), 4, 4, 0, p)),
        (1, lambda: lib.vc_hip_expert_linear_forward(None, p, ctypes.byref(plan), 4, 4, 0, p)),
        (1, lambda: lib.vc_hip_expert_gated_forward(p, p, None, ctypes.byref(plan), 4, 4, 0, p, None, None)),
        (1, lambda: lib.vc_hip_expert_gated_forward(p, p, p, ctypes.byref(plan), 4, 4, 0, p, p, None)),
        (1, lambda: lib.vc_hip_expert_gated_backward(p, p, None, 4, p, p)),
        (1, lambda: lib.vc_hip_expert_linear_backward_input(p, p, p, None, ctypes.byref(plan), 4, 4, p)),
        (1, lambda: lib.vc_hip_expert_linear_backward_input(p, p, None, None, ctypes.byref(plan), 4, 4, None)),
        (1, lambda: lib.vc_hip_expert_linear_backward_weight(p, p, p, ctypes.byref(plan), 4, 4, 0, p, None)),
        (1, lambda: lib.vc_hip_expert_linear_backward_weight(p, None, None, ctypes.byref(plan), 4, 4, 0, p, None)),
        (1, lambda: lib.vc_hip_expert_combine_forward(None, p, ctypes.byref(plan), 4, p)),
        (1, lambda: lib.vc_hip_expert_combine_backward(p, p, None, ctypes.byref(plan), 4, p, None)),
        (1, lambda: lib.vc_hip_orthogonalise(None, 1, 4, 4, 5, p)), (1, lambda: lib.vc_hip_orthogonalise(p, 1 << 20, 4, 4, 5, p)),
        (3, lambda: lib.vc_hip_orthogonalise(p, 1, 1 << 31, 4, 5, p)),
        (1, lambda: lib.vc_hip_muon_step(None, 1, 0.1, 0.9, 0.0, 5)), (1, lambda: lib.vc_hip_muon_step(item(), 1, 0.1, 0.9, 0.0, 0)),
        (1, lambda: lib.vc_hip_muon_step(item(grad=None), 1, 0.1, 0.9, 0.0, 5)),
        (3, lambda: lib.vc_hip_muon_step(item(rows=1 << 31), 1, 0.1, 0.9, 0.0, 5)),
        (1, lambda: lib.vc_hip_when_done(C.WHEN_DONE(), None)), (1, lambda: lib.vc_hip_stream(None)),
    ]


def test_without_a_device():
    if C.available():
        pytest.skip("a GPU is present; covered by the gpu test")
    lib = C.lib()
    for status, call in calls(lib, 16):
        assert call() in (status, 5)  # 5: VC_HIP_ERR_UNAVAILABLE
        assert lib.vc_hip_last_error()


@pytest.mark.gpu
def test_statuses_and_messages():
    lib = C.lib()
    p = ctypes.c_void_p()
    C.check(lib.vc_hip_alloc(4096, ctypes.byref(p)))
    try:
        for i, (status, call) in enumerate(calls(lib, p.value)):
            assert call() == status, i
            assert lib.vc_hip_last_error()
        # Nothing to do is no error.
        plan = C.ExpertPlan(p.value, 0, 2, 8)
        C.check(lib.vc_hip_route_forward(None, None, 0, 8, 2, 0, 1, 1, 1, None, None))
        C.check(lib.vc_hip_expert_linear_forward(None, None, ctypes.byref(plan), 4, 4, 0, None))
        C.check(lib.vc_hip_orthogonalise(None, 0, 4, 4, 5, None))
        C.check(lib.vc_hip_muon_step(None, 0, 0.1, 0.9, 0.0, 5))
        C.synchronize()
    finally:
        C.check(lib.vc_hip_release(p))
