"""Checks of recorded work, kept knowledge and memory that another library writes: a result keeps the values that its operands had when
it was asked for, once the work asked for is synchronised with the other library's write. test_shared_memory.py runs them;
torch is imported first, so that the process has one HIP runtime."""

import gc
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import vectorcore_amd as vc  # noqa: E402

N = 48


def whole(seed, *shape):
    """Small whole numbers: their products and sums are exact in any order."""
    return np.random.default_rng(seed).integers(-4, 5, shape).astype(np.float32)


def overwrite(*tensors):
    """What a caller does before writing shared memory: the work asked for here is done, then the write is."""
    vc.synchronize()
    for t in tensors:
        t.fill_(77.0)
    if tensors[0].is_cuda:
        torch.cuda.synchronize()


def results(x, w, b):
    """Name: result, of operations that may be recorded and computed later, which read x, w or b."""
    other = vc.Tensor(whole(9, N, N), device=x.device)
    return {"left": x @ other, "right": other @ w, "both": x @ w, "layer": other @ w + b, "bias": other @ other + b,
            "relu": (x @ w + b).relu(), "late relu": (other @ other + b).relu()}


def wanted(x, w, b):
    o = whole(9, N, N)
    return {"left": x @ o, "right": o @ w, "both": x @ w, "layer": o @ w + b, "bias": o @ o + b,
            "relu": np.maximum(x @ w + b, 0), "late relu": np.maximum(o @ o + b, 0)}


def elementwise(x, w):
    """The same of elementwise operations whose operands want gradients."""
    half = vc.Tensor(np.full((N, N), 0.5, np.float32), device=x.device)
    return {"add": x + w, "chain": (x * 2.0 + w) * half - x, "one": x * 3.0, "rows": (x * w).sum(1), "columns": (x * w).sum(0),
            "relu": (x - w).relu(), "mean": (x * 2.0).mean()}


def elementwise_wanted(x, w):
    return {"add": x + w, "chain": (x * 2 + w) * 0.5 - x, "one": x * 3, "rows": (x * w).sum(1), "columns": (x * w).sum(0),
            "relu": np.maximum(x - w, 0), "mean": (x * 2).astype(np.float64).mean()}


def compare(got, want):
    for name in want:
        np.testing.assert_allclose(got[name].numpy(), want[name], rtol=2.0 ** -23, atol=0, err_msg=name)


def inputs(torch_device):
    x, w, b = whole(1, N, N), whole(2, N, N), whole(3, N)
    return (x, w, b), [torch.tensor(a, device=torch_device) for a in (x, w, b)]


def check_results_of_imported_memory(device, torch_device):
    host, shared = inputs(torch_device)
    x, w, b = vc.from_dlpack(*shared)
    got = results(x, w, b)
    overwrite(*shared)
    compare(got, wanted(*host))
    compare(results(x, w, b), wanted(*(np.full_like(a, 77) for a in host)))  # what is asked for now reads what is there now


def check_elementwise_results_of_imported_memory(device, torch_device):
    host, shared = inputs(torch_device)
    x, w, _ = vc.from_dlpack(*shared)
    x.requires_grad = w.requires_grad = True
    got = elementwise(x, w)
    overwrite(*shared)
    compare(got, elementwise_wanted(*host[:2]))


def check_results_recorded_before_an_export(device, torch_device):
    host, _ = inputs(torch_device)
    x, w, b = (vc.Tensor(a, device=device) for a in host)
    got = results(x, w, b)
    leaves = [vc.Tensor(a, device=device, requires_grad=True) for a in host[:2]]
    more = elementwise(*leaves)
    shared = [torch.from_dlpack(t.detach()) for t in (x, w, b, *leaves)]
    overwrite(*shared)
    compare(got, wanted(*host))
    compare(more, elementwise_wanted(*host[:2]))


def check_results_of_exported_memory(device, torch_device):
    host, _ = inputs(torch_device)
    x, w, b = (vc.Tensor(a, device=device) for a in host)
    shared = [torch.from_dlpack(t) for t in (x, w, b)]
    got = results(x, w, b)
    overwrite(*shared)
    compare(got, wanted(*host))
    # The other library lets go: nothing else writes the memory, and steps here keep what was recorded.
    del shared
    gc.collect()
    got = results(x, w, b)
    was = [t.numpy() for t in (x, w, b)]
    vc.muon_step([x, w], [vc.Tensor.zeros((N, N), device=device) for _ in range(2)], 0.1,
                 grads=[vc.Tensor(whole(5, N, N), device=device)] * 2)
    compare(got, wanted(*was))
    assert (x.numpy() != was[0]).any()


def check_softmax_gradients(device, torch_device):
    """The rule reads the operand as it was, also where another library writes it before the backward pass."""
    values, up = np.random.default_rng(4).standard_normal((2, 70, 33)).astype(np.float32)
    for log in (False, True):
        def gradient(x, between):
            x.requires_grad = True
            y = x.log_softmax(1) if log else x.softmax(1)
            between()
            y.backward(vc.Tensor(up, device=device))
            return x.grad.numpy()
        want = gradient(vc.Tensor(values, device=device), lambda: None)
        t = torch.tensor(values, device=torch_device)
        np.testing.assert_array_equal(gradient(vc.from_dlpack(t)[0], lambda: overwrite(t)), want)
        q = vc.Tensor(values, device=device)
        np.testing.assert_array_equal(gradient(q, lambda: overwrite(torch.from_dlpack(q.detach()))), want)


def check_gradients_of_a_pass_that_fails(device, torch_device):
    """Gradients that a failing backward pass had stored already."""
    seed = torch.tensor(whole(6, N, N), device=torch_device)
    want = whole(6, N, N) * 2.0
    a, b = (vc.Tensor(whole(s, N, N), device=device, requires_grad=True) for s in (7, 8))
    spoilt = b * b
    out = spoilt + a * 2.0
    vc.muon_step([b], [vc.Tensor.zeros((N, N), device=device)], 0.1, grads=[vc.Tensor(whole(5, N, N), device=device)])
    try:
        out.backward(vc.from_dlpack(seed)[0])
        raise AssertionError("the pass read an operand that had changed")
    except RuntimeError as e:
        assert "modified in place" in str(e)
    overwrite(seed)
    np.testing.assert_array_equal(a.grad.numpy(), want)


def check_largest_class_after_a_write(device, torch_device):
    """The loss may keep each row's argmax; after a write from outside it is that of the new values."""
    rows, classes = 40, 23
    targets = list(range(10)) * 4
    first, second = np.random.default_rng(5).standard_normal((2, rows, classes)).astype(np.float32)
    t = torch.tensor(first, device=torch_device)
    x = vc.from_dlpack(t)[0]
    q = vc.Tensor(first, device=device)
    shared = torch.from_dlpack(q)
    for mine, theirs in ((x, t), (q, shared)):
        vc.cross_entropy(mine, targets).item()
        vc.synchronize()
        theirs.copy_(torch.tensor(second))
        if theirs.is_cuda:
            torch.cuda.synchronize()
        np.testing.assert_array_equal(mine.argmax(1).numpy(), second.argmax(1))
    # One exported and let go of between the loss and the argmax.
    q = vc.Tensor(first, device=device)
    vc.cross_entropy(q, targets).item()
    overwrite(torch.from_dlpack(q))
    gc.collect()
    np.testing.assert_array_equal(q.argmax(1).numpy(), np.zeros(rows))


def check_gradients_that_are_the_seed(device, torch_device):
    """Sums and views pass the gradient on as it is: a stored one is no part of the seed's memory."""
    up = whole(6, N, N)
    for lend in (False, True):
        if lend:
            seed = vc.Tensor(up, device=device)
            memory = torch.from_dlpack(seed)
        else:
            memory = torch.tensor(up, device=torch_device)
            seed = vc.from_dlpack(memory)[0]
        a, b, c = (vc.Tensor(whole(s, N, N), device=device, requires_grad=True) for s in (7, 8, 9))
        kept = a + c.reshape([N * N]).reshape([N, N])
        kept.retain_grad()
        (kept + b).backward(seed)
        b.backward(seed)
        overwrite(memory)
        for t, times in ((a, 1), (c, 1), (kept, 1), (b, 2)):
            np.testing.assert_array_equal(t.grad.numpy(), times * up)


def check_numbers_that_are_no_stream(device, torch_device):
    for stream in (-2, "default"):
        try:
            vc.Tensor(np.zeros(3, np.float32), device=device).__dlpack__(stream=stream)
            raise AssertionError("taken")
        except RuntimeError:
            pass


def check_steps_of_overlapping_memory(device, torch_device):
    """Tensors imported apart that lie over the same memory: refused before anything is written, but for gradients."""
    memory = torch.tensor(whole(2, 4 * N), device=torch_device)
    part = lambda begin, count=N: vc.from_dlpack(memory[begin:begin + count].reshape(4, -1))[0]
    apart = lambda: vc.Tensor(whole(3, 4, N // 4), device=device)
    for p, m, g in (([part(0)], [part(0)], [apart()]), ([part(0)], [apart()], [part(0)]), ([apart()], [part(5)], [part(0)]),
                    ([part(0)], [part(N - 1)], [apart()]), ([part(0), part(2 * N), part(N)], [apart(), apart(), apart()], [apart(), apart(), part(3)]),
                    ([apart(), part(0)], [part(8), apart()], [apart(), apart()])):
        before = [t.numpy() for t in p + m]
        try:
            vc.muon_step(p, m, 0.1, grads=g)
            raise AssertionError("taken")
        except ValueError as e:
            assert "overlap" in str(e)
        for t, was in zip(p + m, before):
            np.testing.assert_array_equal(t.numpy(), was)
    p, m = [part(0), part(N)], [apart(), part(3 * N)]
    vc.muon_step(p, m, 0.1, grads=[part(2 * N), part(2 * N)])  # neighbours, and one gradient twice
    np.testing.assert_array_equal(vc.from_dlpack(memory)[0].numpy()[2 * N:3 * N], whole(2, 4 * N)[2 * N:3 * N])
    assert (p[0].numpy() != whole(2, 4 * N)[:N].reshape(4, -1)).any() and (p[1].numpy() != whole(2, 4 * N)[N:2 * N].reshape(4, -1)).any()


def check_steps_of_one_buffer_imported_twice(device, torch_device):
    """Tied weights: every import's update counts, in the order of the list."""
    memory = torch.zeros(40, 50, device=torch_device)
    tied = [vc.from_dlpack(memory)[0] for _ in range(3)]
    part = vc.from_dlpack(memory[3:9])[0]
    own = vc.Tensor(np.zeros((40, 50), np.float32), device=device)
    lent = torch.from_dlpack(own)
    again = vc.from_dlpack(lent)[0]
    params = [tied[0], part, tied[1], own, again, tied[2]]
    for i, p in enumerate(params):
        p.requires_grad = True
        (p * float(2 ** i)).sum().backward()
    vc.sgd_step(params, 1.0)
    want = np.full((40, 50), -(1.0 + 4 + 32))
    want[3:9] -= 2
    np.testing.assert_array_equal(tied[1].numpy(), want)
    np.testing.assert_array_equal(own.numpy(), np.full((40, 50), -(8.0 + 16)))


def check_picks_written_before_the_gradient(device, torch_device):
    """No promise of a gradient's values, but of its bounds: numbers that are no expert's read and write nothing outside."""
    for score in ("softmax", "sigmoid"):
        for renormalise in (False, True):
            logits = vc.Tensor(np.random.default_rng(6).standard_normal((6, 5)).astype(np.float32), requires_grad=True, device=device)
            weights, chosen = vc.route(logits, 2, score=score, renormalise=renormalise)
            vc.synchronize()
            shared = torch.from_dlpack(chosen)
            shared[:, 0] = torch.tensor([-1.0, 5.0, 1e9, float("nan"), float("inf"), 2.0 ** 33])
            if shared.is_cuda:
                torch.cuda.synchronize()
            weights.backward(vc.Tensor(np.ones((6, 2), np.float32), device=device))
            assert np.isfinite(logits.grad.numpy()).all()


def check_negative_views(device, torch_device):
    """torch negates these when it reads them: the memory holds other values."""
    z = torch.tensor([1 + 2j], device=torch_device).conj()
    for view in (z.imag, torch.arange(4.0, device=torch_device)._neg_view()):
        try:
            vc.from_dlpack(view)
            raise AssertionError("taken with the wrong sign")
        except ValueError as e:
            assert "resolve_neg" in str(e)
        np.testing.assert_array_equal(vc.from_dlpack(view.resolve_neg())[0].numpy(), view.resolve_neg().cpu().numpy())


def check_order_of_later_writes():
    """Neither side waits for the host: importing and exporting a tensor again orders what was enqueued since."""
    n = 1 << 22
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            t = torch.zeros(n, device="cuda")
            p = vc.from_dlpack(t)[0]
            p.requires_grad = True
            (p * 3.0).sum().backward()
            m = torch.ones(2048, 2048, device="cuda")
            for i in range(3):
                for _ in range(6):  # keeps torch's stream busy
                    m = (m @ m).clamp(max=1.0)
                before = t + m[0, 0] - 1.0  # read late
                vc.from_dlpack(t)           # the step waits for that
                vc.sgd_step([p], 1.0)
                torch.from_dlpack(p.detach())  # torch waits for the step
                after = t.clone()
                for _ in range(6):
                    m = (m @ m).clamp(max=1.0)
                t.add_(m[0, 0])
                vc.from_dlpack(t)
                late = p.detach() * 2.0
                assert (before == -2.0 * i).all().item()
                assert (after == -2.0 * i - 3.0).all().item()
                assert (late.numpy() == 2 * (-2.0 * i - 2.0)).all()


RECORDED = [check_results_of_imported_memory, check_elementwise_results_of_imported_memory,
            check_results_recorded_before_an_export, check_results_of_exported_memory, check_softmax_gradients,
            check_gradients_of_a_pass_that_fails]
KEPT = [check_largest_class_after_a_write, check_negative_views, check_picks_written_before_the_gradient, check_steps_of_overlapping_memory,
        check_steps_of_one_buffer_imported_twice, check_gradients_that_are_the_seed,
        check_numbers_that_are_no_stream]
GPU = [check_order_of_later_writes]

if __name__ == "__main__":
    failed = []
    for check in RECORDED + KEPT + GPU:
        try:
            check(*(() if check in GPU else ("hip", "cuda")))
            print(check.__name__, "passed", flush=True)
        except AssertionError as e:
            failed.append(check.__name__)
            print(check.__name__, "FAILED", str(e).strip().replace("\n", " ")[:300], flush=True)
    torch.cuda.synchronize()
    vc.synchronize()
    print("all passed" if not failed else "failed", flush=True)
