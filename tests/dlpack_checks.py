"""Checks of memory shared with torch by DLPack: values both ways without a copy, in-place writes, lifetimes, the order of
work across streams, and refusals. test_dlpack.py runs them; torch is imported first, so that the process has one HIP
runtime."""

import gc
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import vectorcore_amd as vc  # noqa: E402


def check_both_ways_share_memory(device, torch_device):
    a = torch.arange(12, dtype=torch.float32, device=torch_device).reshape(3, 4)
    b = torch.ones(5, device=torch_device)
    x, y = vc.from_dlpack(a, b)
    assert x.device == y.device == device and tuple(x.shape) == (3, 4) and not x.requires_grad
    np.testing.assert_array_equal(x.numpy(), np.arange(12, dtype=np.float32).reshape(3, 4))
    back = torch.from_dlpack(x)
    assert back.data_ptr() == a.data_ptr() and back.device.type == torch_device
    out = torch.from_dlpack((x * 2.0).reshape([4, 3]))
    torch.testing.assert_close(out.cpu(), (a * 2).reshape(4, 3).cpu(), rtol=0, atol=0)
    p = vc.from_dlpack(b)[0]
    p.requires_grad = True
    (p * 3.0).sum().backward()
    vc.sgd_step([p], 0.5)
    torch.testing.assert_close(torch.from_dlpack(p.detach()).cpu(), torch.full((5,), -0.5), rtol=0, atol=0)
    vc.synchronize()
    torch.testing.assert_close(b.cpu(), torch.full((5,), -0.5), rtol=0, atol=0)


def check_views_and_small_tensors(device, torch_device):
    a = torch.arange(100, dtype=torch.float32, device=torch_device)
    x = vc.from_dlpack(a[1:8])[0]  # 4 bytes past any alignment
    np.testing.assert_array_equal((x + x).numpy(), 2 * np.arange(1, 8, dtype=np.float32))
    big = torch.randn(515, 131, device=torch_device).reshape(-1)[1:1 + 514 * 131].reshape(514, 131)
    m = vc.from_dlpack(big)[0]
    w = np.random.default_rng(0).standard_normal((131, 67)).astype(np.float32)
    want = big.cpu().double().numpy() @ w.astype(np.float64)
    np.testing.assert_allclose((m @ vc.Tensor(w, device=device)).numpy(), want, rtol=0, atol=2e-4)
    s = vc.Tensor(np.float32(2.5), device=device)  # a value the hip device keeps on the host until it is needed
    t = torch.from_dlpack(s)
    assert t.shape == () and float(t) == 2.5
    t.fill_(4.0)
    if torch_device == "cuda":
        torch.cuda.synchronize()
    assert s.item() == 4.0
    e = vc.from_dlpack(torch.empty(0, 3, device=torch_device))[0]
    assert tuple(e.shape) == (0, 3) and e.numpy().shape == (0, 3)


def check_pending_readers_of_shared_memory(device, torch_device):
    """An in-place step writes the shared memory itself, also while results that read the old values are still pending."""
    a = torch.full((40, 40), 2.0, device=torch_device)
    p = vc.from_dlpack(a)[0]
    p.requires_grad = True
    q = vc.Tensor(np.full((40, 40), 3.0, np.float32), requires_grad=True, device=device)
    q_seen = torch.from_dlpack(q.detach())
    eye = vc.Tensor(np.eye(40, dtype=np.float32), device=device)
    product, total, other = eye @ p, p + eye, eye @ q
    vc.muon_step([p, q], [vc.Tensor.zeros((40, 40), device=device) for _ in range(2)], 1.0,
                 grads=[vc.Tensor(np.eye(40, dtype=np.float32), device=device)] * 2)
    np.testing.assert_array_equal(product.numpy(), np.full((40, 40), 2.0))
    np.testing.assert_array_equal(total.numpy(), np.full((40, 40), 2.0) + np.eye(40))
    np.testing.assert_array_equal(other.numpy(), np.full((40, 40), 3.0))
    vc.synchronize()
    np.testing.assert_array_equal(a.cpu().numpy(), p.numpy())
    np.testing.assert_array_equal(q_seen.cpu().numpy(), q.numpy())
    assert a[0, 0].item() != 2.0 and q_seen[0, 0].item() != 3.0


def check_numpy_and_lifetimes_on_the_host():
    a = np.arange(6, dtype=np.float32)
    x = vc.from_dlpack(a)[0]
    del a
    gc.collect()
    np.testing.assert_array_equal(x.numpy(), np.arange(6))
    t = torch.from_dlpack(x)
    del x
    gc.collect()
    np.testing.assert_array_equal(t.numpy(), np.arange(6))
    assert vc.Tensor(np.zeros(3)).__dlpack_device__() == (1, 0)


def check_refusals(device, torch_device):
    for bad in (torch.zeros(3, dtype=torch.float64, device=torch_device), torch.zeros(3, dtype=torch.int32, device=torch_device),
                torch.zeros(3, 4, device=torch_device).t(), torch.zeros(8, device=torch_device)[::2],
                torch.zeros(3, device=torch_device, requires_grad=True)):
        with pytest.raises(ValueError):
            vc.from_dlpack(bad)
    if device == "hip":  # a device or host is asked for by name
        with pytest.raises(RuntimeError):
            vc.Tensor(np.zeros(3), device=device).__dlpack__(dl_device=(1, 0))
    with pytest.raises(AttributeError):
        vc.from_dlpack([1.0, 2.0])
    x = vc.Tensor(np.zeros(3), requires_grad=True, device=device)
    with pytest.raises(RuntimeError, match="detach"):
        x.__dlpack__()
    with pytest.raises(RuntimeError):
        x.detach().__dlpack__(copy=True)
    assert vc.from_dlpack() == ()


def check_order_of_work_across_streams():
    """Neither side waits for the host: values written late on one side are read on the other."""
    side = torch.cuda.Stream()
    n = 1 << 22
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            m = torch.ones(2048, 2048, device="cuda")
            for i in range(4):
                for _ in range(4):  # keeps the producer's stream busy
                    m = (m @ m).clamp(max=1.0)
                a = torch.full((n,), float(i), device="cuda") * m[0, 0]
                x = vc.from_dlpack(a)[0]
                y = x * 2.0 + x
                b = torch.from_dlpack(y)
                total = (b + a).double().sum().item()
                assert total == 4.0 * i * n


def check_buffers_are_reused_in_order():
    """Memory given up on either side while the other side's work on it is still queued."""
    n = 1 << 22
    results = []
    for i in range(12):
        a = torch.full((n,), float(i), device="cuda")
        x = vc.from_dlpack(a)[0]
        del a  # torch's memory lives until the work here is done
        y = x + 1.0
        for _ in range(3):
            y = y + x
        del x
        b = torch.from_dlpack(y)
        del y
        results.append(b.mul(2.0))  # queued on torch's stream; then the exported buffer goes back to the pool here
        del b
    for i, r in enumerate(results):
        assert (r == 2.0 * (4.0 * i + 1.0)).all().item()


SHARED = [check_both_ways_share_memory, check_views_and_small_tensors, check_pending_readers_of_shared_memory, check_refusals]
HOST = [check_numpy_and_lifetimes_on_the_host]
GPU = [check_order_of_work_across_streams, check_buffers_are_reused_in_order]

if __name__ == "__main__":
    for check in SHARED:
        print(check.__name__, flush=True)
        check("hip", "cuda")
    for check in GPU:
        print(check.__name__, flush=True)
        check()
    torch.cuda.synchronize()
    vc.synchronize()
    print("all passed", flush=True)
