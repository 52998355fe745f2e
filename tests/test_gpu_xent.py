"""Softmax + cross entropy straight from the connected layer's inputs, against the fp64 form.

Tolerances: z is within e_z = (k + 16) * 2^-23 * sum|x w| + roundings of its bias (see test_gpu_connected);
log sum exp moves by at most the largest e_z of the row, and its own sum of n terms in [0, 1] (fp32, at most
256 in a row before tiles are merged) adds a few hundred roundings relative to it; a probability's relative
error is e_z plus lse's; the products take d rounded to 16 bits.
"""
from __future__ import annotations

import pytest
import torch

import plain64 as P
from plain64 import U

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
SHAPES = [  # batch, inputs, classes
    (1, 64, 10), (1, 8, 1), (3, 77, 5), (5, 128, 1000), (64, 72, 255), (65, 64, 257), (130, 200, 2001), (256, 96, 1000),
    (513, 40, 777), (700, 64, 5000), (2049, 72, 2311), (2, 64, 40000),
]


def _make(seed, M, K, N, dtype, ignored=0.0, bias=True, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = n(M, K).to(dtype), (n(N, K) * spread * K ** -0.5).to(dtype)
    labels = torch.randint(0, N, (M,), generator=g, device="cuda", dtype=torch.int32)
    if ignored:
        drop = torch.rand(M, generator=g, device="cuda") < ignored
        labels = torch.where(drop, torch.full_like(labels, -100), labels)
    return x, w, n(N) * 0.5 if bias else None, labels


def _forward(x, w, b, labels, **kw):
    from darknet_zig_b200 import gpu

    (M, K), N = x.shape, w.shape[0]
    loss, lse = torch.full((M,), 9.0, device="cuda"), torch.full((M,), 9.0, device="cuda")
    gpu.connectedXentForward(x, w, b, labels, loss, lse, M, K, N, **kw)
    return loss, lse


def _z_error(x, w, b):
    e = (x.shape[1] + 16) * 2 * U * (x.double().abs() @ w.double().abs().t())
    return e + 2 * U * (e / (2 * U * 16) + b.double().abs()) if b is not None else e


def _lse_error(x, w, b, lse):
    return _z_error(x, w, b).amax(dim=1) + 300 * U + 4 * U * lse.abs()


def _check_forward(x, w, b, labels):
    loss, lse = _forward(x, w, b, labels)
    want_loss, want_lse = P.xent_forward(x, w, b, labels)
    e = _lse_error(x, w, b, want_lse)
    P.assert_within(lse, want_lse, e, "lse")
    P.assert_within(loss, want_loss, 2 * e + 2 * U * want_loss.abs(), "loss")
    pad = (labels < 0) | (labels >= w.shape[0])
    assert (loss[pad] == 0).all() and (lse[pad] == 0).all()
    return loss, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda, shape, dtype):
    _check_forward(*_make(1, *shape, dtype))


@pytest.mark.parametrize("ignored", [0.3, 0.97, 1.0])
@pytest.mark.parametrize("shape", [(70, 64, 300), (1500, 64, 3000)])
def test_forward_padding_rows(cuda, shape, ignored):
    x, w, b, labels = _make(2, *shape, torch.bfloat16, ignored if ignored < 1 else 0.5)
    if ignored == 1.0:
        labels.fill_(shape[2])  # one past the last class
    clean = _check_forward(x, w, b, labels)
    pad = (labels < 0) | (labels >= shape[2])
    x[pad] = float("nan")
    for got, want in zip(_forward(x, w, b, labels), clean):
        assert torch.equal(got, want)


def test_forward_strides(cuda):
    x, w, b, labels = _make(3, 300, 100, 700, torch.float16)
    want = _forward(x, w, b, labels)
    for pad in (1, 4, 8):
        wide = lambda t: torch.cat([t, torch.full((t.shape[0], pad), float("nan"), device="cuda").to(t.dtype)], 1)[:, :t.shape[1]]  # noqa: E731,E501
        for got, same in zip(_forward(wide(x), wide(w), b, labels), want):
            assert torch.equal(got, same)


def test_forward_confident_and_shifted(cuda):
    """A bias common to all classes moves lse and not the loss; a label that has all the probability."""
    x, w, b, labels = _make(4, 40, 64, 500, torch.bfloat16)
    big = b + 1000.0
    loss, lse = _forward(x, w, big, labels)
    want, wl = P.xent_forward(x, w, big, labels)
    P.assert_within(lse, wl, _lse_error(x, w, big, wl), "lse")
    P.assert_within(loss, want, 2 * _lse_error(x, w, big, wl) + 4 * U * 1000, "loss")
    b2 = b.clone()
    b2[labels[0].long()] = 80.0
    loss, _ = _forward(x, w, b2, labels)
    assert loss[0].item() < 1e-4


def test_forward_infinities(cuda):
    x, w, b, labels = _make(5, 20, 64, 300, torch.bfloat16)
    labels[:] = 7
    b[100:200] = float("-inf")  # classes that cannot occur
    _check_forward(x, w, b, labels)
    b[:] = float("-inf")
    b[7] = 0.5
    loss, lse = _forward(x, w, b, labels)
    P.assert_within(loss, torch.zeros(20, device="cuda"), 1e-5, "loss")
    b[:] = float("-inf")
    _, lse = _forward(x, w, b, labels)
    assert (lse == float("-inf")).all()
    b[:] = 0.0
    b[3] = float("inf")
    _, lse = _forward(x, w, b, labels)
    assert (lse == float("inf")).all()
    x[4, 5] = float("nan")
    b[3] = 0.0
    loss, lse = _forward(x, w, b, labels)
    assert torch.isnan(loss[4]) and torch.isnan(lse[4]) and torch.isfinite(loss[5:]).all()


def test_forward_impossible_tile_beside_small_outputs(cuda):
    """A whole tile of classes that cannot occur, and the others far below 0."""
    x, w, b, labels = _make(16, 20, 64, 700, torch.bfloat16)
    labels[:] = 600
    b[:300] = float("-inf")
    b[300:] -= 300.0
    _check_forward(x, w, b, labels)


def _backward(x, w, b, labels, lse, rs, scale, dw_type=None, accumulate=0, want=(1, 1, 1), pad=0, workspace=None):
    from darknet_zig_b200 import gpu

    (M, K), N = x.shape, w.shape[0]
    new = lambda r, c, t: torch.full((r, c + pad), 3.0, device="cuda", dtype=t)  # noqa: E731
    dxb, dwb = new(M, K, x.dtype), new(N, K, dw_type or x.dtype)
    db = torch.full((N,), 2.0, device="cuda")
    gpu.connectedXentBackward(x, w, b, labels, lse, rs, scale, dxb[:, :K] if want[0] else None, db if want[1] else None,
                              dwb[:, :K] if want[2] else None, M, K, N, accumulate=accumulate, workspace=workspace)
    assert (dxb[:, K:] == 3).all() and (dwb[:, K:] == 3).all()
    return dxb[:, :K], dwb[:, :K], db


def _check_backward(x, w, b, labels, rs=None, scale=1.0, **kw):
    accumulate = kw.get("accumulate", 0)
    lse = P.xent_forward(torch.nan_to_num(x), w, b, labels)[1].float()
    dx, dw, db = _backward(x, w, b, labels, lse, rs, scale, **kw)
    wx, ww, wb, d = P.xent_backward(x, w, b, labels, rs, scale)
    x0 = torch.where(((labels >= 0) & (labels < w.shape[0]))[:, None], x.double(), torch.zeros_like(x.double()))
    factor = scale * (rs.double().abs() if rs is not None else torch.ones(x.shape[0], device="cuda", dtype=torch.float64))
    p = torch.softmax(x0 @ w.double().t() + (b.double() if b is not None else 0), dim=1) * factor.abs()[:, None]
    p = torch.where((d != 0).any(dim=1)[:, None], p, torch.zeros_like(p))
    # d before rounding; then its rounding to 16 bits (of d / f * 2^14: subnormal steps of f16 are 2^-38 of f)
    e_d = p * (_z_error(x0, w, b) + _lse_error(x0, w, b, lse.double())[:, None] + 8 * U) + 4 * U * d.abs()
    h = P.half_step(x.dtype)
    e_r = e_d + h * (d.abs() + e_d) + factor.abs()[:, None] * (d != 0) * P.tiny(x.dtype) / 16384
    M, N = d.shape
    add_x, add_w = (3.0 if accumulate & 2 else 0.0), (3.0 if accumulate & 1 else 0.0)
    want = wx + add_x
    tol = e_r @ w.double().abs() + (N + 32) * 2 * U * (d.abs() @ w.double().abs()) + 8 * U * (want.abs() + add_x)
    P.assert_within(dx, want, tol + h * (want.abs() + tol) + P.tiny(x.dtype), "dx")
    want = ww + add_w
    e_x = e_r + (h * d.abs() if rs is not None else 0)  # x times its row's factor is rounded too
    tol = e_x.t() @ x0.abs() + (M + 32) * 2 * U * (d.abs().t() @ x0.abs()) + 8 * U * (want.abs() + add_w)
    hw = P.half_step(dw.dtype)
    P.assert_within(dw, want, tol + hw * (want.abs() + tol) + P.tiny(dw.dtype), "weight_updates")
    add = 2.0 if accumulate & 1 else 0.0
    P.assert_within(db, wb + add, e_d.sum(dim=0) + 40 * U * d.abs().sum(dim=0) + 2 * U * (wb.abs() + add), "bias_updates")
    return dx, dw, db, lse


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(cuda, shape, dtype):
    _check_backward(*_make(6, *shape, dtype), scale=0.25 if dtype == torch.bfloat16 else 8.0)


@pytest.mark.parametrize("ignored", [0.4, 0.97])
@pytest.mark.parametrize("shape", [(70, 64, 300), (1500, 72, 3000)])
@pytest.mark.parametrize("scaled", [False, True])
def test_backward_padding_rows(cuda, shape, ignored, scaled):
    x, w, b, labels = _make(7, *shape, torch.bfloat16, ignored)
    x[(labels < 0)] = float("nan")
    rs = torch.rand(shape[0], device="cuda") + 0.1 if scaled else None
    if scaled:
        rs[labels < 0] = float("inf")
    _check_backward(x, w, b, labels, rs=None if rs is None else torch.nan_to_num(rs, posinf=1.0), accumulate=0)
    if scaled:
        good = _backward(x, w, b, labels, P.xent_forward(torch.nan_to_num(x), w, b, labels)[1].float(), rs, 1.0)
        assert all(torch.isfinite(t).all() for t in good)


def test_backward_all_padding(cuda):
    x, w, b, labels = _make(8, 90, 64, 300, torch.bfloat16)
    labels.fill_(-1)
    lse = torch.zeros(90, device="cuda")
    dx, dw, db = _backward(x, w, b, labels, lse, None, 1.0)
    assert (dx == 0).all() and (dw == 0).all() and (db == 0).all()
    dx, dw, db = _backward(x, w, b, labels, lse, None, 1.0, accumulate=3, dw_type=torch.float32)
    assert (dx == 3).all() and (dw == 3).all() and (db == 2).all()


@pytest.mark.parametrize("accumulate", [0, 1, 2, 3])
@pytest.mark.parametrize("dw_type", [torch.float16, torch.float32])
def test_backward_accumulates(cuda, accumulate, dw_type):
    x, w, b, labels = _make(9, 200, 130, 450, torch.float16, 0.2)
    _check_backward(x, w, b, labels, accumulate=accumulate, dw_type=dw_type, scale=2.0, pad=accumulate)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("accumulate", [0, 3])
def test_backward_in_pieces(cuda, dtype, accumulate):
    """More classes than one piece holds (65536 rows make a piece 2048 classes wide)."""
    x, w, b, labels = _make(10, 65600, 24, 4500, dtype, 0.1)
    rs = torch.rand(65600, device="cuda") * 2 - 0.5
    _check_backward(x, w, b, labels, rs=rs, scale=0.01 if dtype == torch.bfloat16 else 1.0, accumulate=accumulate)


def test_backward_wide_row_scales(cuda):
    """Factors far apart and far from 1: each row's dx keeps its own relative precision."""
    x, w, b, labels = _make(11, 64, 64, 200, torch.float16)
    rs = torch.logspace(-3, 3, 64, device="cuda") * 1e-1
    _check_backward(x, w, b, labels, rs=rs)


def test_backward_parts(cuda):
    x, w, b, labels = _make(12, 300, 64, 900, torch.bfloat16, 0.1)
    lse = _forward(x, w, b, labels)[1]
    dx, dw, db = _backward(x, w, b, labels, lse, None, 0.5)
    assert torch.equal(_backward(x, w, b, labels, lse, None, 0.5, want=(1, 0, 0))[0], dx)
    assert torch.equal(_backward(x, w, b, labels, lse, None, 0.5, want=(0, 1, 0))[2], db)
    assert torch.equal(_backward(x, w, b, labels, lse, None, 0.5, want=(0, 0, 1))[1], dw)


def test_gradient_against_differences(cuda):
    """Minus the loss's slope along a direction: fp64 differences of the plain loss at the kernel's inputs, h
    small enough that the third derivative's h^2 term is below the 16-bit deltas' own rounding."""
    x, w, b, labels = _make(13, 30, 64, 100, torch.float16)
    lse = _forward(x, w, b, labels)[1]
    dx, dw, db = _backward(x, w, b, labels, lse, None, 1.0, dw_type=torch.float32)
    g = torch.Generator(device="cuda").manual_seed(1)
    for at, grad in ((x, dx), (w, dw), (b, db)):
        v = torch.randn(at.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        f = lambda s: P.xent_forward(*(t.double() + s * v if t is at else t.double() for t in (x, w, b)), labels)[0].sum()  # noqa: E731,E501
        slope = (f(h) - f(-h)) / (2 * h)
        along = (grad.double() * v).sum()
        # d's and dx's roundings, worst case: 2 half steps of the terms' magnitudes
        bound = 2 * P.half_step(x.dtype) * (grad.double().abs() * v.abs()).sum() + 1e-3 * slope.abs() + 1e-3
        assert abs(along + slope) <= bound


def test_repeatable_and_captured(cuda):
    x, w, b, labels = _make(14, 1000, 200, 3000, torch.bfloat16, 0.2)
    loss, lse = _forward(x, w, b, labels)
    first = _backward(x, w, b, labels, lse, None, 0.1)
    for _ in range(3):
        for got, same in zip(_forward(x, w, b, labels), (loss, lse)):
            assert torch.equal(got, same)
        for got, same in zip(_backward(x, w, b, labels, lse, None, 0.1), first):
            assert torch.equal(got, same)
    from darknet_zig_b200 import gpu

    out = [torch.empty(1000, device="cuda"), torch.empty(1000, device="cuda")]
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(3000, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu.connectedXentForward(x, w, b, labels, *out, 1000, 200, 3000)
        gpu.connectedXentBackward(x, w, b, labels, out[1], None, 0.1, dx, db, dw, 1000, 200, 3000, accumulate=0)
    x2, w2, _, labels2 = _make(15, 1000, 200, 3000, torch.bfloat16, 0.6)
    x.copy_(x2)
    w.copy_(w2)
    labels.copy_(labels2)
    graph.replay()
    loss, lse = _forward(x, w, b, labels)
    want = _backward(x, w, b, labels, lse, None, 0.1)
    for got, same in zip(out + [dx, dw, db], [loss, lse, *want]):
        assert torch.equal(got, same)


def test_one_training_run(cuda):
    """The set together, as a step uses it: group norm on channels-last, a 1x1 convolution with residual, the
    loss and its deltas, back through both, and the mixed update; against the fp64 forms fed with the
    kernels' own 16-bit intermediates, each within its own tolerance elsewhere: here the run's plumbing is
    checked (which tensor goes where, in which sign) by the loss falling along the updates' direction in fp64."""
    from darknet_zig_b200 import gpu

    B, S, C, N, G = 4, 49, 64, 100, 8
    M = B * S
    g = torch.Generator(device="cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, sc, bi = n(B, S, C).bfloat16(), torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    w1f, w2f = n(C, C) * C ** -0.5, n(N, C) * C ** -0.5
    w1, w2 = w1f.bfloat16(), w2f.bfloat16()
    labels = torch.randint(0, N, (M,), generator=g, device="cuda", dtype=torch.int32)
    h, z = torch.empty_like(x), torch.empty(M, C, device="cuda", dtype=torch.bfloat16)
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    gpu.gnActForward(x, h, B, S, C, G, sc, bi, 1e-5, mean, rstd, P.LEAKY)
    gpu.connectedActForward(h, w1, None, x, z, M, C, C, P.LEAKY)
    gpu.connectedXentForward(z, w2, None, labels, loss, lse, M, C, N)
    dz, dh, dx = torch.empty_like(z), torch.empty_like(z), torch.empty_like(x)
    u1, u2 = torch.zeros(C, C, device="cuda"), torch.zeros(N, C, device="cuda")
    bu, su = torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    gpu.connectedXentBackward(z, w2, None, labels, lse, None, 1.0, dz, None, u2, M, C, N)
    gpu.connectedActBackward(h, w1, z, dz, dz, dh, None, u1, M, C, C, P.LEAKY)
    gpu.gnActBackward(x, h, dh.view(B, S, C), dx, B, S, C, G, sc, bi, mean, rstd, bu, su, P.LEAKY)
    dx = dx.double() + dz.double().view(B, S, C)  # the residual's delta is dz

    def f(x_, sc_, bi_, w1_, w2_):
        a = P.gn_forward(x_, G, sc_, bi_, 1e-5, P.LEAKY)[0].reshape(M, C)
        y = P.connected_forward(a, w1_, None, x_.reshape(M, C), P.LEAKY)
        return P.xent_forward(y, w2_, None, labels)[0].sum()

    at = [t.double() for t in (x, sc, bi, w1, w2)]
    base = f(*at)
    # loss: three 16-bit roundings of values of order one, each 2^-9 of them through slopes below 2, over M rows
    assert abs(base - loss.double().sum()) <= M * 3 * 2 * 2 ** -9
    for i, u in enumerate((dx, su, bu, u1, u2)):
        # step so that the first-order change is 1e-3 of the loss's scale; then second order is far below it
        size = (u.double() ** 2).sum()
        step = 1e-3 / size.sqrt()
        moved = [t + step * u.double() if j == i else t for j, t in enumerate(at)]
        fall, first = base - f(*moved), step * size
        # the slope along u is -|u|^2 for the exact deltas; 16-bit deltas are within a few 2^-9 in norm per
        # stage and leaky's sign may differ where an intermediate rounds to the other side: 10 % covers both
        assert abs(fall - first) <= 0.1 * first, (i, fall.item(), first.item())
    v1, w16 = torch.zeros_like(u1), torch.empty_like(w1)
    before, change = w1f.clone(), 0.1 / M * u1
    want = before + change
    gpu.sgdMomentumMixed(w1f, u1, None, w16, C, C, 0.1, 0.9, 0.0, M)
    # w + a*u: the factor a = lr/batch is rounded on each side (2 U), a*u once more in `want` (1 U), each sum
    # once (2 U of a result below |w| + |a*u|); relative to the summands, for the sum may cancel
    P.assert_within(w1f, want, 5 * U * (before.abs() + change.abs()), "weights")
    assert torch.equal(w16, w1f.bfloat16()) and (v1 == 0).all()


def test_no_device_error(cuda):
    from darknet_zig_b200 import gpu

    gpu.check_device_error()
