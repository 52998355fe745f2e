"""The fp64 backward formulas the GPU tests compare with, against central differences of the forward ones
(an error of O(h^2) from the third derivative and O(2^-53 / h) from rounding: 1e-6 relative covers both at
h = 1e-5 with values of order one)."""
from __future__ import annotations

import pytest
import torch

import plain64 as P


def _differences(f, a, h=1e-5):
    out = torch.zeros_like(a)
    flat, res = a.view(-1), out.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + h
        up = f()
        flat[i] = keep - h
        down = f()
        flat[i] = keep
        res[i] = (up - down) / (2 * h)
    return out


def _gen(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("name", ["linear", "leaky", "logistic", "tanh"])
@pytest.mark.parametrize("groups", [1, 2, 6])
def test_gn_backward_formula(name, groups):
    n, a = _gen(1), P.ACTS[name]
    x, sc, bi, delta = n(2, 3, 6), n(6), n(6), n(2, 3, 6)
    loss = lambda: (P.gn_forward(x, groups, sc, bi, 1e-5, a)[0] * delta).sum()  # noqa: E731
    mean, rstd = P.gn_stats(x, groups, 1e-5)
    dx, db, ds, _ = P.gn_backward(x, None, delta, groups, sc, bi, mean, rstd, a)
    for got, at in ((dx, x), (db, bi), (ds, sc)):
        torch.testing.assert_close(got, _differences(loss, at), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("name", ["linear", "leaky", "logistic", "relu"])
def test_connected_backward_formula(name):
    n, a = _gen(2), P.ACTS[name]
    x, w, b, r, delta = n(3, 5), n(4, 5), n(4), n(3, 4), n(3, 4)
    loss = lambda: (P.connected_forward(x, w, b, r, a) * delta).sum()  # noqa: E731
    dz, dx, dw, db = P.connected_backward(x, w, P.connected_forward(x, w, b, r, a), delta, a)
    for got, at in ((dz, r), (dx, x), (dw, w), (db, b)):
        torch.testing.assert_close(got, _differences(loss, at), rtol=1e-6, atol=1e-6)


def test_xent_backward_formula():
    """Deltas are minus the gradient of scale * sum(row_scales * loss) (darknet: truth - prediction)."""
    n = _gen(3)
    x, w, b, rs = n(4, 5), n(7, 5), n(7), n(4)
    labels = torch.tensor([3, -1, 0, 6], dtype=torch.int32)
    loss = lambda: -0.7 * (P.xent_forward(x, w, b, labels)[0] * rs).sum()  # noqa: E731
    dx, dw, db, _ = P.xent_backward(x, w, b, labels, rs, 0.7)
    for got, at in ((dx, x), (dw, w), (db, b)):
        torch.testing.assert_close(got, _differences(loss, at), rtol=1e-6, atol=1e-6)
