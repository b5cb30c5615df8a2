"""Dropout against its definition: the generator's published test vectors, which elements are kept, exact values, residuals,
infinities in dropped places, gradients, and refusals."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]


def philox(block, stream, seed):
    """Philox 4x32 with ten rounds on Python's integers."""
    low = 0xFFFFFFFF
    c, k = [block & low, block >> 32, stream & low, stream >> 32], [seed & low, seed >> 32]
    for _ in range(10):
        first, second = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(second >> 32) ^ c[1] ^ k[0], second & low, (first >> 32) ^ c[3] ^ k[1], first & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def words(count, seed, stream):
    return np.array([w for b in range((count + 3) // 4) for w in philox(b, stream, seed)][:count], np.uint64)


def expected(x, p, seed, stream=0, residual=None):
    kept = (words(x.size, seed, stream) >= round(p * 2 ** 32)).reshape(x.shape)
    with np.errstate(over="ignore"):
        y = np.where(kept, x * np.float32(1 / (1 - p)), np.float32(0))
    return y if residual is None else y + residual


def test_the_generator_here_is_the_published_one():
    """Known answers of the generator's authors (Random123, kat_vectors: philox4x32 10)."""
    assert philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox(2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    counter, key = (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)
    assert philox(counter[0] | counter[1] << 32, counter[2] | counter[3] << 32, key[0] | key[1] << 32) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("count", [1, 2, 3, 4, 5, 7, 255, 256, 257, 1023, 4099, 20001])
@pytest.mark.parametrize("joined", [False, True])
def test_values_are_exact(count, joined, device):
    rng = np.random.default_rng(count)
    x, r, dy = (rng.standard_normal(count).astype(np.float32) for _ in range(3))
    seed, stream = 2 ** 63 + count, 2 ** 40 + 7
    tx, tr = vc.Tensor(x, requires_grad=True, device=device), vc.Tensor(r, requires_grad=True, device=device)
    y = vc.dropout(tx, 0.3, seed, stream=stream, residual=tr if joined else None)
    y.backward(vc.Tensor(dy, device=device))
    np.testing.assert_array_equal(y.numpy(), expected(x, 0.3, seed, stream, r if joined else None))
    np.testing.assert_array_equal(tx.grad.numpy(), expected(dy, 0.3, seed, stream))
    if joined:
        np.testing.assert_array_equal(tr.grad.numpy(), dy)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("p", [2.0 ** -33, 2.0 ** -32, 0.1, 0.5, 0.9, 1 - 2.0 ** -32])
def test_borders_of_the_words(p, device):
    """The element whose word is the threshold is kept, the one just below it is not."""
    seed = 11
    w = words(64, seed, 0)
    x = np.ones(64, np.float32)
    for i in (0, 5, 63):
        at = float(w[i]) / 2 ** 32
        assert vc.dropout(vc.Tensor(x, device=device), at, seed).numpy()[i] == np.float32(1 / (1 - at))
        assert vc.dropout(vc.Tensor(x, device=device), at + 2.0 ** -32, seed).numpy()[i] == 0
    np.testing.assert_array_equal(vc.dropout(vc.Tensor(x, device=device), p, seed).numpy(), expected(x, p, seed))


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_and_everything(device):
    x = np.array([1.0, -np.inf, np.nan, 3.0, 2.0], np.float32)
    r = np.arange(5, dtype=np.float32)
    t = lambda v, grad=False: vc.Tensor(v, requires_grad=grad, device=device)
    np.testing.assert_array_equal(vc.dropout(t(x), 0.0, 1).numpy(), x)
    np.testing.assert_array_equal(vc.dropout(t(x), 0.0, 1, residual=t(r)).numpy(), x + r)
    np.testing.assert_array_equal(vc.dropout(t(x), 1.0, 1).numpy(), np.zeros(5, np.float32))
    np.testing.assert_array_equal(vc.dropout(t(x), 1.0, 1, residual=t(r)).numpy(), r)
    tx = t(r, True)
    vc.dropout(tx, 1.0, 1).sum().backward()
    np.testing.assert_array_equal(tx.grad.numpy(), np.zeros(5, np.float32))
    tx, tr = t(r, True), t(r, True)
    vc.dropout(tx, 0.0, 1, residual=tr).sum().backward()
    np.testing.assert_array_equal(tx.grad.numpy(), np.ones(5, np.float32))
    np.testing.assert_array_equal(tr.grad.numpy(), np.ones(5, np.float32))


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_dropped_does_not_matter(device):
    """Infinities and NaN in dropped places, of x and of the upstream gradient."""
    x = np.linspace(-2, 2, 1001).astype(np.float32)
    clean = expected(x, 0.5, 3)
    dirty = x.copy()
    dropped = np.flatnonzero(words(1001, 3, 0) < 2 ** 31)
    dirty[dropped] = np.resize(np.array([np.inf, -np.inf, np.nan], np.float32), len(dropped))
    np.testing.assert_array_equal(vc.dropout(vc.Tensor(dirty, device=device), 0.5, 3).numpy(), clean)
    tx = vc.Tensor(x, requires_grad=True, device=device)
    vc.dropout(tx, 0.5, 3).backward(vc.Tensor(dirty, device=device))
    np.testing.assert_array_equal(tx.grad.numpy(), clean)


@pytest.mark.parametrize("device", DEVICES)
def test_streams_and_seeds_differ_and_shapes_do_not(device):
    x = np.ones((40, 50), np.float32)
    run = lambda v, seed, stream=0: vc.dropout(vc.Tensor(v, device=device), 0.5, seed, stream=stream).numpy()
    first = run(x, 1)
    np.testing.assert_array_equal(first.ravel(), run(x.reshape(10, 200), 1).ravel())
    np.testing.assert_array_equal(first, run(x, 1))
    for other in (run(x, 2), run(x, 1 + 2 ** 32), run(x, 1, 1), run(x, 1, 2 ** 32)):
        # Two independent masks of 2000 elements agree in 1000 +- 22.4 of them: eight deviations.
        assert abs((first == other).sum() - 1000) < 180


@pytest.mark.parametrize("device", DEVICES)
def test_shares_and_the_same_tensor_twice(device):
    x = np.ones(40000, np.float32)
    for p in (0.1, 0.75):
        kept = (vc.dropout(vc.Tensor(x, device=device), p, 99).numpy() != 0).mean()
        assert abs(kept - (1 - p)) < 8 * (p * (1 - p) / 40000) ** 0.5
    tx = vc.Tensor(x[:9], requires_grad=True, device=device)
    vc.dropout(tx, 0.5, 4, residual=tx).sum().backward()
    np.testing.assert_array_equal(tx.grad.numpy(), 1 + expected(x[:9], 0.5, 4))
    assert tuple(vc.dropout(vc.Tensor(np.ones((0, 3), np.float32), device=device), 0.5, 1).shape) == (0, 3)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = vc.Tensor(np.ones((2, 3), np.float32), device=device)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            vc.dropout(x, p, 1)
    for bad in ((3, 2), (3,), (2, 1)):
        with pytest.raises(ValueError):
            vc.dropout(x, 0.5, 1, residual=vc.Tensor(np.ones(bad, np.float32), device=device))
    with pytest.raises(TypeError):
        vc.dropout(x, 0.5)
    with pytest.raises(TypeError):
        vc.dropout(x, 0.5, -1)
    if device == "hip":
        with pytest.raises(ValueError, match="expected hip"):
            vc.dropout(x, 0.5, 1, residual=vc.Tensor(np.ones((2, 3), np.float32)))
