"""SGD on fp32 weights with 16-bit gradients in and 16-bit weights out: the fp32 results are bit-exact
against dnb_axpy / dnb_scal's arithmetic (one fused rounding each), the 16-bit copy is the weights rounded."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _fma(a, b, c):
    """a*b + c rounded once: a*b is exact in fp64 and the sum's second rounding differs from one rounding
    only in double-rounding ties, which the comparison allows one ulp for."""
    return np.float32(np.float64(a) * b.astype(np.float64) + c.astype(np.float64))


def _rows(t, pad):
    out = torch.full((t.shape[0], t.shape[1] + pad), 7.0, device="cuda", dtype=t.dtype)
    out[:, :t.shape[1]] = t
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols,pad_g,pad_w", [
    (1, 1, 0, 0), (1, 7, 0, 3), (5, 8, 0, 0), (5, 8, 8, 16), (33, 1023, 0, 1), (33, 1023, 1, 0), (64, 100, 0, 0),
    (300, 72, 8, 0), (3, 4099, 5, 5), (1000, 1024, 0, 0), (1, 100003, 0, 0)])
def test_update(cuda, dtype, rows, cols, pad_g, pad_w):
    from darknet_zig_b200 import gpu

    g = torch.Generator(device="cuda").manual_seed(rows * cols)
    n = lambda: torch.randn(rows, cols, generator=g, device="cuda")  # noqa: E731
    w, wu, gr = n(), n(), n().to(dtype)
    w0, wu0 = w.cpu().numpy(), wu.cpu().numpy()
    gbuf, wbuf = _rows(gr, pad_g), _rows(torch.zeros_like(gr), pad_w)
    lr, mom, decay, batch = 0.01, 0.9, 5e-4, 16
    for use_g in (True, False):
        w.copy_(torch.from_numpy(w0))
        wu.copy_(torch.from_numpy(wu0))
        gpu.sgdMomentumMixed(w, wu, gbuf[:, :cols] if use_g else None, wbuf[:, :cols], rows, cols, lr, mom, decay,
                             batch)
        u = wu0 + gr.float().cpu().numpy() if use_g else wu0
        u = _fma(np.float32(-np.float32(decay) * np.float32(batch)), w0, u)
        want_w = _fma(np.float32(lr) / np.float32(batch), u, w0)
        want_u = u * np.float32(mom)
        got_w, got_u = w.cpu().numpy(), wu.cpu().numpy()
        # one ulp where the emulated fma rounded twice
        assert np.all(np.abs(got_w - want_w) <= np.spacing(np.abs(want_w)) * 1)
        assert np.all(np.abs(got_u - want_u) <= np.spacing(np.abs(want_u)) * 2)
        assert torch.equal(wbuf[:, :cols], w.to(dtype))
        assert (wbuf[:, cols:] == 7.0).all() and (gbuf[:, cols:] == 7.0).all()


def test_gradients_may_be_the_weights16(cuda):
    from darknet_zig_b200 import gpu

    w, wu = torch.randn(16, 64, device="cuda"), torch.zeros(16, 64, device="cuda")
    g = torch.randn(16, 64, device="cuda").bfloat16()
    a, b, out = w.clone(), wu.clone(), torch.empty_like(g)
    gpu.sgdMomentumMixed(a, b, g, out, 16, 64, 0.1, 0.9, 0.0, 4)
    gpu.sgdMomentumMixed(w, wu, g, g, 16, 64, 0.1, 0.9, 0.0, 4)
    assert torch.equal(a, w) and torch.equal(b, wu) and torch.equal(out, g)


def test_agrees_with_the_fp32_update(cuda):
    """Without gradients the fp32 results are dnb_sgd_momentum's, bit for bit."""
    from darknet_zig_b200 import gpu

    w, wu = torch.randn(77, 91, device="cuda"), torch.randn(77, 91, device="cuda")
    a, b, out = w.clone(), wu.clone(), torch.empty(77, 91, device="cuda", dtype=torch.float16)
    gpu.sgdMomentum(77 * 91, w, wu, 0.05, 0.9, 1e-4, 32)
    gpu.sgdMomentumMixed(a, b, None, out, 77, 91, 0.05, 0.9, 1e-4, 32)
    assert torch.equal(a, w) and torch.equal(b, wu) and torch.equal(out, w.half())
