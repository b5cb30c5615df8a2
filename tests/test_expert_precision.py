"""The expert products at float32's precision: errors against float64 next to those of the same products in float32.
Operands of two bfloat16 parts (16 bits) would not pass."""

import numpy as np
import pytest

import vectorcore_amd as vc

DEVICES = ["cpu", pytest.param("hip", marks=pytest.mark.gpu)]
UNIT = 2.0 ** -24
SIZES = [(2, 40, 70), (30, 64, 33), (70, 33, 80), (300, 96, 131), (300, 36, 260), (2500, 80, 96)]


def norm(x):
    return np.sqrt((x * x).sum())


def products(x, w, g):
    """y = x w and the gradients g w^T and x^T g."""
    return x @ w, g @ w.T, x.T @ g


def limits(x, w, g):
    """Eight times the error of the same products in float32, and two roundings of the result. Three bfloat16 parts hold all
    of a value and the products left out are 2^-26 of the largest, so a term costs a quarter of a rounding more; the six
    products' sums in float32 round up to six times where a float32 chain rounds once a term, in sums of sixteen terms."""
    exact = products(*(a.astype(np.float64) for a in (x, w, g)))
    return exact, [8 * norm(a - b) + 2 * UNIT * norm(b) for a, b in zip(products(x, w, g), exact)]


def operands(rows, width, columns):
    rng = np.random.default_rng(rows + width)
    return [rng.standard_normal(s).astype(np.float32) for s in ((rows, width), (width, columns), (rows, columns))]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,width,columns", SIZES)
def test_error_is_that_of_float32(rows, width, columns, device):
    x, w, g = operands(rows, width, columns)
    plan = vc.ExpertPlan(vc.Tensor(np.zeros((rows, 1), np.float32), device=device), 1)
    tx, tw = vc.Tensor(x, requires_grad=True, device=device), vc.Tensor(w[None], requires_grad=True, device=device)
    y = vc.expert_linear(tx, tw, plan)
    y.backward(vc.Tensor(g, device=device))
    exact, most = limits(x, w, g)
    for got, want, limit in zip((y.numpy(), tx.grad.numpy(), tw.grad.numpy()[0]), exact, most):
        assert norm(got - want) <= limit
    # The gated unit, whose two products and their own product are held against the same in float32.
    up = w[:, ::-1].copy()
    h = vc.expert_gated(vc.Tensor(x, device=device), vc.Tensor(w[None], device=device), vc.Tensor(up[None], device=device), plan)
    a, b = x.astype(np.float64) @ w, x.astype(np.float64) @ up
    limit = 8 * norm((x @ w) / (1 + np.exp(-(x @ w))) * (x @ up) - a / (1 + np.exp(-a)) * b) + 2 * UNIT * norm(a / (1 + np.exp(-a)) * b)
    assert norm(h.numpy() - a / (1 + np.exp(-a)) * b) <= limit


def two_parts(v):
    """The nearest sum of two bfloat16 numbers, near enough."""
    def bfloat16(a):
        bits = a.astype(np.float32).view(np.uint32)
        return ((bits + 0x7FFF + (bits >> 16 & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    first = bfloat16(v)
    return first.astype(np.float64) + bfloat16(v - first)


@pytest.mark.parametrize("rows,width,columns", SIZES)
def test_two_parts_would_not_pass(rows, width, columns):
    """The bound tells three parts from two, even where everything else is exact: products of short sums at least."""
    x, w, g = operands(rows, width, columns)
    exact, most = limits(x, w, g)
    worst = [norm(a - b) / limit for a, b, limit in zip(products(*map(two_parts, (x, w, g))), exact, most)]
    assert max(worst) > 1.5
