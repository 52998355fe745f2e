"""Where the 16-bit entries write: inside the workspace they ask for, and at offsets beyond 32 bits."""
from __future__ import annotations

import ctypes

import pytest
import torch

import plain64 as P

pytestmark = pytest.mark.gpu
CANARY = 0xA5


def _exact(name, *args):
    """A workspace of exactly the bytes the query names, and the canary bytes behind it."""
    from darknet_zig_b200 import gpu

    n = ctypes.c_size_t(0)
    gpu.call(name + "_workspace", *args, ctypes.byref(n))
    buf = torch.full((n.value + 4096,), CANARY, dtype=torch.uint8, device="cuda")
    return buf[:n.value], buf[n.value:]


def _ptr(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("shape", [(2, 20000, 64, 1), (1, 9000, 24, 2), (3, 49, 64, 8), (2, 391, 330, 33)])
def test_gn_workspaces(cuda, shape):
    from darknet_zig_b200 import gpu

    B, S, C, G = shape
    x, delta = torch.randn(B, S, C, device="cuda").bfloat16(), torch.randn(B, S, C, device="cuda").bfloat16()
    y, dx = torch.empty_like(x), torch.empty_like(x)
    sc, bi = torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    mean, rstd = torch.empty(B, G, device="cuda"), torch.empty(B, G, device="cuda")
    ws, tail = _exact("gn_act_forward", _ptr(x), _ptr(y), gpu.BF16, B, S, C, G)
    gpu.gnActForward(x, y, B, S, C, G, sc, bi, 1e-5, mean, rstd, P.LEAKY, workspace=ws)
    assert (tail == CANARY).all()
    ws, tail = _exact("gn_act_backward", _ptr(x), _ptr(y), _ptr(delta), _ptr(dx), gpu.BF16, B, S, C, G)
    gpu.gnActBackward(x, y, delta, dx, B, S, C, G, sc, bi, mean, rstd, sc.clone(), bi.clone(), P.LEAKY, workspace=ws)
    assert (tail == CANARY).all()


@pytest.mark.parametrize("shape", [(1, 33, 7), (40, 301, 99), (777, 1023, 1000), (2100, 73, 2401)])
def test_product_workspaces(cuda, shape):
    from darknet_zig_b200 import gpu

    M, K, N = shape
    x, w = torch.randn(M, K, device="cuda").half(), torch.randn(N, K, device="cuda").half()
    y, delta = torch.empty(M, N, device="cuda").half(), torch.randn(M, N, device="cuda").half()
    ws, tail = _exact("connected_act_forward", _ptr(x), K, _ptr(w), K, gpu.F16, M, K, N)
    gpu.connectedActForward(x, w, None, None, y, M, K, N, P.LEAKY, workspace=ws)
    assert (tail == CANARY).all()
    dz, dx, dw = torch.empty_like(y), torch.empty_like(x), torch.empty_like(w)
    ws, tail = _exact("connected_act_backward", _ptr(x), K, _ptr(w), K, _ptr(delta), N, _ptr(dz), N, gpu.F16, M, K, N,
                      P.LEAKY)
    gpu.connectedActBackward(x, w, y, delta, dz, dx, torch.empty(N, device="cuda"), dw, M, K, N, P.LEAKY, 0, workspace=ws)
    assert (tail == CANARY).all()
    labels = torch.randint(-1, N, (M,), device="cuda", dtype=torch.int32)
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    ws, tail = _exact("connected_xent_forward", _ptr(x), K, _ptr(w), K, gpu.F16, M, K, N)
    gpu.connectedXentForward(x, w, None, labels, loss, lse, M, K, N, workspace=ws)
    assert (tail == CANARY).all()
    ws, tail = _exact("connected_xent_backward", _ptr(x), K, _ptr(w), K, gpu.F16, M, K, N)
    gpu.connectedXentBackward(x, w, None, labels, lse, torch.rand(M, device="cuda"), 1.0, dx,
                              torch.empty(N, device="cuda"), dw, M, K, N, 0, workspace=ws)
    assert (tail == CANARY).all()


@pytest.mark.parametrize("M", [2, 5])
def test_rows_beyond_32_bit_offsets(cuda, M):
    """Rows 2^30 elements apart: the last one starts beyond 2^31 bytes, and from M = 5 on beyond 2^32 elements."""
    from darknet_zig_b200 import gpu

    K, N, ld = 192, 136, 1 << 30
    flat = torch.empty(ld * (M - 1) + 256, device="cuda", dtype=torch.bfloat16)
    x = flat.as_strided((M, K), (ld, 1))
    x.copy_(torch.randn(M, K, device="cuda"))
    w = torch.randn(N, K, device="cuda").bfloat16()
    y, near = torch.empty(M, N, device="cuda").bfloat16(), torch.empty(M, N, device="cuda").bfloat16()
    gpu.connectedActForward(x, w, None, None, y, M, K, N, P.LEAKY)
    gpu.connectedActForward(x.contiguous(), w, None, None, near, M, K, N, P.LEAKY)
    assert torch.equal(y, near)
    out = flat.as_strided((M, N), (ld, 1))
    xc = x.contiguous()
    gpu.connectedActForward(xc, w, None, None, out, M, K, N, P.LEAKY)
    assert torch.equal(out.contiguous(), near)
