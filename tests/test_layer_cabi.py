"""Refusals of the C entry points of layer normalisation, dropout and the loss of a linear layer: a status and a message,
nothing launched."""

import ctypes

import pytest

from vectorcore_amd import cabi as C


def calls(lib, p):
    """(status code, call) pairs; p: a device pointer that no refused call reads."""
    inf, nan = float("inf"), float("nan")
    return [
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 0, 1e-5, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 4, -1.0, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 4, nan, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 4, inf, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(None, None, None, 3, 4, 1e-5, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 4, 1e-5, None, None)),
        (1, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 4, 1e-5, p, p + 4)),
        (3, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 3, 1 << 30, 1e-5, p, None)),
        (3, lambda: lib.vc_hip_layer_norm_forward(p, None, None, 1 << 50, 4, 1e-5, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_backward(None, p, None, p, 3, 4, p, None, None)),
        (1, lambda: lib.vc_hip_layer_norm_backward(p, None, None, p, 3, 4, p, None, None)),
        (1, lambda: lib.vc_hip_layer_norm_backward(p, p, None, None, 3, 4, None, p, None)),
        (1, lambda: lib.vc_hip_layer_norm_backward(p, p, None, p + 4, 3, 4, None, None, p)),
        (1, lambda: lib.vc_hip_layer_norm_backward(p, p, None, p, 3, 0, p, None, None)),
        (3, lambda: lib.vc_hip_layer_norm_backward(p, p, None, p, 1 << 45, 4, p, None, None)),
        (1, lambda: lib.vc_hip_dropout(p, None, 4, -0.5, 1, 0, p)), (1, lambda: lib.vc_hip_dropout(p, None, 4, 1.5, 1, 0, p)),
        (1, lambda: lib.vc_hip_dropout(p, None, 4, nan, 1, 0, p)), (1, lambda: lib.vc_hip_dropout(None, None, 4, 0.5, 1, 0, p)),
        (1, lambda: lib.vc_hip_dropout(p, p, 4, 0.5, 1, 0, None)), (3, lambda: lib.vc_hip_dropout(p, p, 1 << 50, 0.5, 1, 0, p)),
        (1, lambda: lib.vc_hip_linear_xent_forward(p, p, None, p, 3, 0, 5, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_forward(p, p, None, p, 3, 4, 0, p, None)),
        (3, lambda: lib.vc_hip_linear_xent_forward(p, p, None, p, 3, 4, (1 << 24) + 1, p, None)),
        (3, lambda: lib.vc_hip_linear_xent_forward(p, p, None, p, 1 << 31, 4, 5, p, None)),
        (3, lambda: lib.vc_hip_linear_xent_forward(p, p, None, p, 3, 1 << 25, 5, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_forward(None, p, None, p, 3, 4, 5, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_forward(p, None, None, p, 3, 4, 5, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_forward(p, p, None, None, 3, 4, 5, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_gradient(p, p, None, p, p, 3, 4, 5, p, p, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_gradient(p, p, None, p, None, 3, 0, 5, p, p, p, None)),
        (1, lambda: lib.vc_hip_linear_xent_gradient(None, p, None, p, None, 3, 4, 5, p, p, p, None)),
        (3, lambda: lib.vc_hip_linear_xent_gradient(p, p, None, p, None, 3, 4, 1 << 25, p, p, p, None)),
    ]


def test_without_a_device():
    if C.available():
        pytest.skip("a GPU is present; covered by the gpu test")
    lib = C.lib()
    for status, call in calls(lib, 16):
        assert call() in (status, 5)  # 5: VC_HIP_ERR_UNAVAILABLE
        assert lib.vc_hip_last_error()


@pytest.mark.gpu
def test_on_a_device():
    lib = C.lib()
    p = ctypes.c_void_p()
    assert lib.vc_hip_alloc(256, ctypes.byref(p)) == 0
    try:
        for i, (status, call) in enumerate(calls(lib, p.value)):
            assert call() == status, i
            assert lib.vc_hip_last_error()
        # Nothing asked for, and nothing to do.
        assert lib.vc_hip_layer_norm_backward(None, None, None, None, 3, 4, None, None, None) == 0
        assert lib.vc_hip_layer_norm_forward(None, None, None, 0, 4, 1e-5, None, None) == 0
        assert lib.vc_hip_dropout(None, None, 0, 0.5, 1, 0, None) == 0
        assert lib.vc_hip_linear_xent_forward(None, None, None, None, 0, 4, 5, None, None) == 0
    finally:
        lib.vc_hip_release(p)
    assert lib.vc_hip_synchronize() == 0
