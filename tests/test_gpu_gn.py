"""Group norm + activation, channels last, against the fp64 form.

Tolerances (u = 2^-24): with k terms added in fp32 by a thread (at most `spatial` of them), a sum's error is
at most k*u times the sum of its terms' magnitudes; the fp64 sums on top are exact beside that.
"""
from __future__ import annotations

import pytest
import torch

import plain64 as P
from plain64 import U

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5
pytestmark = pytest.mark.gpu


def _make(seed, B, S, C, dtype, mean=0.3, std=1.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return ((n(B, S, C) * std + mean).to(dtype), n(C) * 0.3 + 1, n(C) * 0.2, n(B, S, C).to(dtype))


def _forward(x, groups, sc, bi, a, eps=EPS, y=None):
    from darknet_zig_b200 import gpu

    B, S, C = x.shape
    y = torch.empty_like(x) if y is None else y
    mean, rstd = torch.empty(B, groups, device="cuda"), torch.empty(B, groups, device="cuda")
    gpu.gnActForward(x, y, B, S, C, groups, sc, bi, eps, mean, rstd, a)
    return y, mean, rstd


def _z_error(x, mean, rstd, sc, bi, k):
    """How far scale*(x - mean)*rstd + bias may be off: the mean to u|mean| plus its sum's error, the
    deviation's and the products' roundings, rstd from a variance with relative error (k + 8)u (halved by
    the square root)."""
    xa = x.double().abs()
    dev = (mean.abs() + xa) * 2 * U + (k + 2) * U * xa.amax()
    xh = ((x.double() - mean) * rstd).abs()
    return sc.double().abs() * (dev * rstd + xh * (k + 8) * U) + 3 * U * (sc.double().abs() * xh + bi.double().abs())


def _check_forward(x, groups, sc, bi, a, eps=EPS):
    B, S, C = x.shape
    y, mean, rstd = _forward(x, groups, sc, bi, a, eps)
    want, wm, wr = P.gn_forward(x, groups, sc, bi, eps, a)
    k = S
    amax = x.double().abs().amax()
    P.assert_within(mean, wm, (k + 2) * U * amax + 1e-37, "mean")
    # var's error: k u relative from the squares, and twice the deviations' error against their spread
    P.assert_within(rstd, wr, wr * (k + 8) * U + wr * (2 * U * amax * wr) * 4, "rstd")
    per = C // groups
    z = _z_error(x, P._wide(wm, per), P._wide(wr, per), sc, bi, k)
    # the activations' slopes are at most 1; logistic and tanh add a few roundings of values below 1
    P.assert_within(y, want, z + 8 * U + P.half_step(x.dtype) * (want.abs() + z) + P.tiny(x.dtype), "y")
    return y, mean, rstd


SHAPES = [  # batch, spatial, filters, groups
    (1, 1, 8, 2), (1, 1, 64, 64), (2, 7, 6, 3), (3, 49, 64, 8), (1, 49, 1024, 32), (2, 391, 330, 33), (2, 64, 33, 11),
    (5, 100, 48, 1), (4, 33, 40, 5), (1, 3, 4096, 1), (2, 5, 8192, 4), (1, 4096, 64, 2), (1, 5000, 320, 32),
    (2, 784, 256, 32), (1, 20000, 64, 1), (1, 9000, 24, 2), (40, 9, 512, 32), (1, 600, 4095, 1), (300, 16, 16, 2),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda, shape, dtype):
    B, S, C, G = shape
    x, sc, bi, _ = _make(1, B, S, C, dtype)
    _check_forward(x, G, sc, bi, P.LEAKY)


@pytest.mark.parametrize("name", sorted(P.ACTS))
def test_forward_activations(cuda, name):
    x, sc, bi, _ = _make(2, 3, 50, 96, torch.bfloat16)
    _check_forward(x, 12, sc, bi, P.ACTS[name])


def test_forward_large_mean(cuda):
    x, sc, bi, _ = _make(3, 2, 400, 64, torch.float32, mean=1000.0, std=0.5)
    _check_forward(x, 8, sc, bi, P.LINEAR)


def test_forward_constant_group_gives_the_bias(cuda):
    x, sc, bi, _ = _make(4, 2, 30, 32, torch.float32)
    x[1, :, 8:16] = 2.5  # exact in fp32: the mean is exact and the deviations are 0
    y, mean, rstd = _forward(x, 4, sc, bi, P.LINEAR)
    assert torch.equal(y[1, :, 8:16], bi[8:16].expand(30, 8))
    assert mean[1, 1].item() == 2.5


def test_forward_in_place_and_repeatable(cuda):
    for shape in ((2, 391, 330, 33), (2, 784, 256, 32), (1, 20000, 64, 1), (1, 4096, 64, 2)):
        B, S, C, G = shape
        x, sc, bi, _ = _make(5, B, S, C, torch.bfloat16)
        y, mean, rstd = _forward(x, G, sc, bi, P.LEAKY)
        for _ in range(3):
            y2, m2, r2 = _forward(x, G, sc, bi, P.LEAKY)
            assert torch.equal(y, y2) and torch.equal(mean, m2) and torch.equal(rstd, r2)
        z = x.clone()
        _forward(z, G, sc, bi, P.LEAKY, y=z)
        assert torch.equal(z, y)


def test_bad_values_stay_in_their_group(cuda):
    for shape in ((2, 391, 330, 33), (1, 20000, 64, 2)):
        B, S, C, G = shape
        x, sc, bi, delta = _make(6, B, S, C, torch.float32)
        clean, cm, cr = _forward(x, G, sc, bi, P.LEAKY)
        x[0, 5, 0] = float("nan")
        y, mean, rstd = _forward(x, G, sc, bi, P.LEAKY)
        per = C // G
        assert torch.isnan(y[0, :, :per]).all() and torch.isnan(mean[0, 0]) and torch.isnan(rstd[0, 0])
        assert torch.equal(y[0, :, per:], clean[0, :, per:]) and torch.equal(y[1:], clean[1:])


def _backward(x, y, delta, groups, sc, bi, mean, rstd, a, accumulate=0, dx=None, bu=None, su=None):
    from darknet_zig_b200 import gpu

    B, S, C = x.shape
    dx = torch.empty_like(x) if dx is None else dx
    bu = torch.full((C,), float("nan"), device="cuda") if bu is None else bu
    su = torch.full((C,), float("nan"), device="cuda") if su is None else su
    gpu.gnActBackward(x, y, delta, dx, B, S, C, groups, sc, bi, mean, rstd, bu, su, a, accumulate=accumulate)
    return dx, bu, su


def _check_backward(x, y, delta, groups, sc, bi, a):
    B, S, C = x.shape
    mean, rstd = (t.float() for t in P.gn_stats(x, groups, EPS))
    dx, bu, su = _backward(x, y, delta, groups, sc, bi, mean, rstd, a)
    want, wb, ws, p = P.gn_backward(x, y, delta, groups, sc, bi, mean, rstd, a)
    k = S + 8
    # xh: the deviation's rounding and the product's; d: the gradient's roundings, and for a recomputed output
    # (slope of act' at most 2 for tanh) its error
    e_xh = (x.double().abs() + p["mean"].abs()) * p["rstd"] * U + p["xh"].abs() * 2 * U
    e_z = sc.double().abs() * e_xh + 3 * U * ((sc.double() * p["xh"]).abs() + bi.double().abs()) + 8 * U
    e_d = p["d"].abs() * 4 * U + delta.double().abs() * (4 * U + (0.0 if y is not None else 2.0) * e_z * (a != P.LINEAR))
    e_t = e_d * sc.double().abs() + p["t"].abs() * U
    per = C // groups
    gm = lambda v: P._wide(v.reshape(B, S, groups, per).mean(dim=(1, 3)), per)  # noqa: E731
    e_m0 = p["a0"] * k * U + gm(e_t)
    e_m1 = p["a1"] * k * U + gm(e_t * p["xh"].abs() + p["t"].abs() * e_xh)
    tol = p["rstd"] * (e_t + e_m0 + p["xh"].abs() * e_m1 + e_xh * p["m1"].abs() +
                       4 * U * (p["t"].abs() + p["m0"].abs() + (p["xh"] * p["m1"]).abs()))
    P.assert_within(dx, want, tol + P.half_step(x.dtype) * (want.abs() + tol) + P.tiny(x.dtype), "dx")
    P.assert_within(bu, wb, (p["d"].abs() * k * U + e_d).sum(dim=(0, 1)) + wb.abs() * U, "bias_updates")
    P.assert_within(su, ws, ((p["d"] * p["xh"]).abs() * k * U + e_d * p["xh"].abs() + p["d"].abs() * e_xh)
                    .sum(dim=(0, 1)) + ws.abs() * U, "scale_updates")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_recomputed(cuda, shape, dtype):
    B, S, C, G = shape
    x, sc, bi, delta = _make(7, B, S, C, dtype)
    _check_backward(x, None, delta, G, sc, bi, P.LOGISTIC)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_from_the_output(cuda, shape, dtype):
    B, S, C, G = shape
    x, sc, bi, delta = _make(8, B, S, C, dtype)
    y, _, _ = _forward(x, G, sc, bi, P.LEAKY)
    _check_backward(x, y, delta, G, sc, bi, P.LEAKY)


@pytest.mark.parametrize("name", sorted(P.ACTS))
def test_backward_activations(cuda, name):
    x, sc, bi, delta = _make(9, 3, 50, 96, torch.bfloat16)
    y, _, _ = _forward(x, 12, sc, bi, P.ACTS[name])
    _check_backward(x, y, delta, 12, sc, bi, P.ACTS[name])


def test_recomputed_output_has_the_forwards_sign(cuda):
    """fp32: the output recomputed in the backward is the forward's, so a kinked activation's gradient is
    the same with and without y."""
    for shape in ((2, 391, 330, 33), (1, 20000, 64, 1), (3, 49, 64, 8)):
        B, S, C, G = shape
        x, sc, bi, delta = _make(10, B, S, C, torch.float32)
        y, mean, rstd = _forward(x, G, sc, bi, P.LEAKY)
        a = _backward(x, y, delta, G, sc, bi, mean, rstd, P.LEAKY)
        b = _backward(x, None, delta, G, sc, bi, mean, rstd, P.LEAKY)
        # the unit cut may differ with the third tensor, and with it the order of the sums: (S + 8)u of the
        # terms' magnitudes covers any order
        _, _, _, p = P.gn_backward(x, y, delta, G, sc, bi, mean, rstd, P.LEAKY)
        P.assert_within(b[1], a[1], 2 * (S + 8) * U * p["d"].abs().sum(dim=(0, 1)), "bias_updates")
        tol = p["rstd"] * 2 * (S + 8) * U * (p["a0"] + p["xh"].abs() * p["a1"]) + a[0].double().abs() * 4 * U
        P.assert_within(b[0], a[0], tol, "dx")


def test_backward_accumulates_in_place(cuda):
    B, S, C, G = 3, 100, 64, 8
    x, sc, bi, delta = _make(11, B, S, C, torch.bfloat16)
    mean, rstd = (t.float() for t in P.gn_stats(x, G, EPS))
    dx, bu, su = _backward(x, None, delta, G, sc, bi, mean, rstd, P.LOGISTIC)
    b2, s2 = torch.ones(C, device="cuda"), torch.full((C,), -2.0, device="cuda")
    d2 = delta.clone()
    _backward(x, None, d2, G, sc, bi, mean, rstd, P.LOGISTIC, accumulate=1, dx=d2, bu=b2, su=s2)
    assert torch.equal(d2, dx)
    P.assert_within(b2, bu.double() + 1, 2 * U * (bu.double().abs() + 1), "bias_updates")
    P.assert_within(s2, su.double() - 2, 2 * U * (su.double().abs() + 2), "scale_updates")


def test_empty(cuda):
    sc = torch.ones(8, device="cuda")
    x = torch.empty(0, 5, 8, device="cuda", dtype=torch.bfloat16)
    _forward(x, 2, sc, sc, P.LEAKY)
    bu, su = torch.full((8,), 3.0, device="cuda"), torch.full((8,), 4.0, device="cuda")
    none = torch.empty(0, 2, device="cuda")
    _backward(x, None, x, 2, sc, sc, none, none, P.LEAKY, accumulate=1, bu=bu, su=su)
    assert (bu == 3).all() and (su == 4).all()
    _backward(x, None, x, 2, sc, sc, none, none, P.LEAKY, accumulate=0, bu=bu, su=su)
    assert (bu == 0).all() and (su == 0).all()


def test_streams_and_graphs(cuda):
    """A captured forward and backward replay on new inputs, from another stream than the capture's."""
    B, S, C, G = 2, 784, 256, 32
    x, sc, bi, delta = _make(12, B, S, C, torch.bfloat16)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    bu, su = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")

    def step():
        from darknet_zig_b200 import gpu

        gpu.gnActForward(x, y, B, S, C, G, sc, bi, EPS, mean, rstd, P.LEAKY)
        gpu.gnActBackward(x, y, delta, dx, B, S, C, G, sc, bi, mean, rstd, bu, su, P.LEAKY, accumulate=0)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    x2, _, _, d2 = _make(13, B, S, C, torch.bfloat16)
    x.copy_(x2)
    delta.copy_(d2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    got = [t.clone() for t in (y, dx, bu, su)]
    step()
    for a, b in zip(got, (y, dx, bu, su)):
        assert torch.equal(a, b)
