"""The connected layer on 16-bit tensors against the fp64 form.

Tolerances: the accumulators are fp32 and each of the k additions may lose up to a whole step (the tensor
core need not round to nearest), so a product is within (k + 16) * 2^-23 of the sum of its terms' magnitudes;
the epilogue adds a few roundings of what it adds, and the result is rounded once to its type.
"""
from __future__ import annotations

import pytest
import torch

import plain64 as P
from plain64 import U

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
SHAPES = [  # batch, inputs, outputs
    (1, 1, 1), (1, 64, 3), (1, 4096, 1000), (2, 77, 130), (3, 1023, 77), (4, 512, 4096), (5, 8, 8), (5, 1, 9),
    (7, 63, 65), (16, 256, 2048), (33, 40, 200), (64, 64, 64), (130, 200, 250), (128, 1024, 129), (777, 1023, 1000),
    (2100, 72, 2400), (300, 4099, 8), (2305, 136, 2303), (9, 70000, 24),
]


def _matrix(g, rows, cols, dtype, pad, std=1.0):
    buf = torch.full((rows, cols + pad), 5.0, device="cuda", dtype=dtype)
    buf[:, :cols] = torch.randn(rows, cols, generator=g, device="cuda") * std
    return buf[:, :cols]


def _product_error(a, b, k):
    return (k + 16) * 2 * U * (a.double().abs() @ b.double().abs())


def _make(seed, M, K, N, dtype, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (_matrix(g, M, K, dtype, pad), _matrix(g, N, K, dtype, pad, max(K, 1) ** -0.5),
            torch.randn(N, generator=g, device="cuda"), _matrix(g, M, N, dtype, pad), _matrix(g, M, N, dtype, pad))


def _forward(x, w, b, r, a, pad=0, y=None, **kw):
    from darknet_zig_b200 import gpu

    (M, K), N = x.shape, w.shape[0]
    buf = torch.full((M, N + pad), 9.0, device="cuda", dtype=x.dtype)
    out = buf[:, :N] if y is None else y
    gpu.connectedActForward(x, w, b, r, out, M, K, N, a, **kw)
    assert (buf[:, N:] == 9.0).all(), "wrote between the rows"
    return out


def _check_forward(x, w, b, r, a, pad=0):
    got = _forward(x, w, b, r, a, pad)
    want = P.connected_forward(x, w, b, r, a)
    tol = _product_error(x, w.t(), x.shape[1])
    mag = want.abs() if a == P.LINEAR else P.connected_forward(x, w, b, r, P.LINEAR).abs()
    tol = tol + 4 * U * (mag + (b.double().abs() if b is not None else 0) + (r.double().abs() if r is not None else 0))
    tol = tol + 8 * U  # logistic, tanh
    P.assert_within(got, want, tol + P.half_step(x.dtype) * (want.abs() + tol) + P.tiny(x.dtype), "y")
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda, shape, dtype):
    x, w, b, r, _ = _make(1, *shape, dtype)
    _check_forward(x, w, b, r, P.LEAKY)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("shape", [(1, 300, 40), (4, 64, 100), (40, 300, 100), (2100, 72, 2400)])
def test_forward_strides(cuda, shape, pad):
    x, w, b, r, _ = _make(2, *shape, torch.bfloat16, pad)
    _check_forward(x, w, b, None, P.LINEAR, pad)
    _check_forward(x, w, None, r, P.RELU, pad)


@pytest.mark.parametrize("name", sorted(P.ACTS))
@pytest.mark.parametrize("M", [1, 50])
def test_forward_activations(cuda, name, M):
    x, w, b, r, _ = _make(3, M, 96, 72, torch.float16)
    _check_forward(x, w, b, r, P.ACTS[name])
    _check_forward(x, w, None, None, P.ACTS[name])


@pytest.mark.parametrize("M", [3, 200])
def test_forward_misaligned_base(cuda, M):
    """Operands whose first row is off a 16-byte boundary although their stride is a whole number of them."""
    g = torch.Generator(device="cuda").manual_seed(4)
    flat = lambda rows, cols, off: torch.randn(rows * 128 + 8, generator=g, device="cuda").half()[off:off + rows * 128].view(rows, 128)[:, :cols]  # noqa: E731,E501
    for off in (1, 4):
        x, w = flat(M, 120, off), flat(60, 120, off)
        _check_forward(x, w, None, None, P.LINEAR)


@pytest.mark.parametrize("M", [1, 4, 300])
def test_forward_into_the_residual(cuda, M):
    x, w, b, r, _ = _make(5, M, 128, 136, torch.bfloat16)
    want = _forward(x, w, b, r, P.RELU)
    r2 = r.clone()
    _forward(x, w, b, r2, P.RELU, y=r2)
    assert torch.equal(r2, want)


def test_forward_without_inputs(cuda):
    for M in (1, 30):
        x, w, b, r, _ = _make(6, M, 0, 16, torch.bfloat16)
        got = _forward(x, w, b, r, P.LINEAR)
        assert torch.equal(got, (b + r.float()).bfloat16())
        assert (_forward(x, w, None, None, P.LOGISTIC) == 0.5).all()


def test_forward_bad_values_stay_in_their_rows(cuda):
    x, w, b, _, _ = _make(7, 300, 200, 150, torch.bfloat16)
    clean = _forward(x, w, b, None, P.LINEAR)
    x[17, 3], x[200, 0] = float("nan"), float("inf")
    got = _forward(x, w, b, None, P.LINEAR)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[17] = keep[200] = False
    assert torch.equal(got[keep], clean[keep])
    assert torch.isnan(got[17]).all() and not torch.isfinite(got[200]).any()


def _backward(x, w, y, delta, a, want_dz=True, dw_type=None, accumulate=0, pad=0, **into):
    from darknet_zig_b200 import gpu

    (M, K), N = x.shape, w.shape[0]
    new = lambda r, c, t: torch.full((r, c + pad), 3.0, device="cuda", dtype=t)[:, :c]  # noqa: E731
    dz = into.get("dz", new(M, N, x.dtype) if a != P.LINEAR else None)
    dx = into.get("dx", new(M, K, x.dtype))
    dw = into.get("dw", new(N, K, dw_type or x.dtype))
    db = into.get("db", torch.full((N,), 2.0, device="cuda"))
    gpu.connectedActBackward(x, w, y if a != P.LINEAR else None, delta, dz, dx, db, dw, M, K, N, a,
                             accumulate=accumulate)
    return dz, dx, dw, db


def _check_backward(x, w, y, delta, a, dw_type=None, accumulate=0, pad=0):
    (M, K), N = x.shape, w.shape[0]
    dz, dx, dw, db = _backward(x, w, y, delta, a, dw_type=dw_type, accumulate=accumulate, pad=pad)
    exact = P.connected_backward(x, w, y, delta, a)
    h, t = P.half_step(x.dtype), P.tiny(x.dtype)
    if a == P.LINEAR:
        dz = delta
    else:
        P.assert_within(dz, exact[0], (4 * U + h) * exact[0].abs() + 4 * U * delta.double().abs() + t, "dz")
    # the products take the rounded dz
    add_x, add_w = (3.0 if accumulate & 2 else 0.0), (3.0 if accumulate & 1 else 0.0)
    want = dz.double() @ w.double() + add_x
    tol = _product_error(dz, w, N) + 4 * U * (want.abs() + add_x)
    P.assert_within(dx, want, tol + h * (want.abs() + tol) + t, "dx")
    want = dz.double().t() @ x.double() + add_w
    tol = _product_error(dz.t(), x, M) + 4 * U * (want.abs() + add_w)
    hw = P.half_step(dw.dtype)
    P.assert_within(dw, want, tol + hw * (want.abs() + tol) + P.tiny(dw.dtype), "weight_updates")
    # fp32 sums of at most 64 rows, then fp64
    add = 2.0 if accumulate & 1 else 0.0
    mag = (delta.double() * P.act_gradient(y.double(), a)).abs() if a != P.LINEAR else delta.double().abs()
    P.assert_within(db, exact[3] + add, ((mag + (a != P.LINEAR) * delta.double().abs()) * 72 * U).sum(dim=0) +
                    2 * U * (exact[3].abs() + add), "bias_updates")


def _outputs(seed, M, N, dtype, a, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = _matrix(g, M, N, dtype, pad)
    y.copy_(P.act(y.double(), a))
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(cuda, shape, dtype):
    x, w, _, _, delta = _make(8, *shape, dtype)
    y = _outputs(9, shape[0], shape[2], dtype, P.LEAKY)
    _check_backward(x, w, y, delta, P.LEAKY)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("a", [P.LINEAR, P.RELU])
def test_backward_strides_and_fp32_updates(cuda, pad, a):
    for shape in ((40, 300, 100), (2100, 72, 2400), (1000, 2050, 2305)):
        x, w, _, _, delta = _make(10, *shape, torch.bfloat16, pad)
        y = _outputs(11, shape[0], shape[2], torch.bfloat16, a, pad)
        _check_backward(x, w, y, delta, a, dw_type=torch.float32, pad=pad)


@pytest.mark.parametrize("accumulate", [1, 2, 3])
def test_backward_accumulates(cuda, accumulate):
    x, w, _, _, delta = _make(12, 200, 130, 96, torch.float16)
    y = _outputs(13, 200, 96, torch.float16, P.LOGISTIC)
    for t in (torch.float16, torch.float32):
        _check_backward(x, w, y, delta, P.LOGISTIC, dw_type=t, accumulate=accumulate)


@pytest.mark.parametrize("name", sorted(P.ACTS))
def test_backward_activations(cuda, name):
    a = P.ACTS[name]
    x, w, _, _, delta = _make(14, 50, 96, 72, torch.bfloat16)
    _check_backward(x, w, _outputs(15, 50, 72, torch.bfloat16, a), delta, a)


def test_backward_in_place_and_parts(cuda):
    """dz may be delta; what is not asked for is not needed."""
    x, w, _, _, delta = _make(16, 100, 64, 80, torch.bfloat16)
    y = _outputs(17, 100, 80, torch.bfloat16, P.LEAKY)
    dz, dx, dw, db = _backward(x, w, y, delta, P.LEAKY)
    d2 = delta.clone()
    z2, x2, w2, b2 = _backward(x, w, y, d2, P.LEAKY, dz=d2)
    assert torch.equal(d2, dz) and torch.equal(x2, dx) and torch.equal(w2, dw) and torch.equal(b2, db)
    _, x3, _, _ = _backward(x, w, y, delta, P.LEAKY, dw=None, db=None)
    _, _, w3, _ = _backward(x, w, y, delta, P.LEAKY, dx=None, db=None)
    _, _, _, b3 = _backward(x, w, y, delta, P.LEAKY, dx=None, dw=None)
    assert torch.equal(x3, dx) and torch.equal(w3, dw) and torch.equal(b3, db)


def test_backward_of_nothing(cuda):
    for accumulate in (0, 3):
        x, w, _, _, delta = _make(18, 0, 16, 8, torch.bfloat16)
        _, dx, dw, db = _backward(x, w, None, delta, P.LINEAR, accumulate=accumulate, dw_type=torch.float32)
        assert (dw == (3.0 if accumulate else 0.0)).all() and (db == (2.0 if accumulate else 0.0)).all()
        x, w, _, _, delta = _make(19, 6, 16, 0, torch.bfloat16)
        _, dx, dw, db = _backward(x, w, None, delta, P.LINEAR, accumulate=accumulate)
        assert (dx == (3.0 if accumulate else 0.0)).all()


def test_repeatable_and_captured(cuda):
    """The same bits every time, eagerly, from a graph, and from two streams at once with a workspace each."""
    x, w, b, r, delta = _make(20, 1000, 1021, 1200, torch.bfloat16)
    y = _forward(x, w, b, r, P.LEAKY)
    first = _backward(x, w, y, delta, P.LEAKY)
    for _ in range(3):
        assert torch.equal(_forward(x, w, b, r, P.LEAKY), y)
        for p, q in zip(_backward(x, w, y, delta, P.LEAKY), first):
            assert torch.equal(p, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = _forward_only(x, w, b, r)
        outs = _backward(x, w, yg, delta, P.LEAKY)
    graph.replay()
    assert torch.equal(yg, y)
    for p, q in zip(outs, first):
        assert torch.equal(p, q)
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([_forward_only(x, w, b, r) for _ in range(4)])
    torch.cuda.synchronize()
    for group in got:
        for t in group:
            assert torch.equal(t, y)


def _forward_only(x, w, b, r):
    from darknet_zig_b200 import gpu

    y = torch.empty(x.shape[0], w.shape[0], device="cuda", dtype=x.dtype)
    gpu.connectedActForward(x, w, b, r, y, x.shape[0], x.shape[1], w.shape[0], P.LEAKY)
    return y


def test_no_device_error(cuda):
    from darknet_zig_b200 import gpu

    gpu.check_device_error()
