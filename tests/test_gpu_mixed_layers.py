"""The 16-bit layers (layers.GroupNorm, layers.Connected) and the loss as a training step uses them: the same
results as the entries they call, and gradients against the fp64 forms at the layers' own values."""
from __future__ import annotations

import pytest
import torch

import plain64 as P
from plain64 import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [P.LEAKY, P.LOGISTIC])
def test_a_block_and_its_update(cuda, act):
    from darknet_zig_b200 import gpu, layers

    torch.manual_seed(5)
    B, S, C, N, G = 3, 25, 64, 90, 8
    M = B * S
    norm, conv = layers.GroupNorm(B, S, C, G, act), layers.Connected(M, C, C, P.RELU)
    head = layers.Connected(M, C, N, P.LINEAR)
    x = torch.randn(B, S, C, device="cuda").bfloat16()
    labels = torch.randint(0, N, (M,), device="cuda", dtype=torch.int32)
    labels[7] = -1
    h = norm.forward(x)
    y = conv.forward(h.view(M, C), x.view(M, C))
    loss, lse = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")
    gpu.connectedXentForward(y, head.weights16, head.biases, labels, loss, lse, M, C, N)
    want, _ = P.xent_forward(y, head.weights16, head.biases, labels)
    P.assert_within(loss, want, 1e-4 * (1 + want.abs()), "loss")  # far above k u |x||w| = 80 * 1.2e-7 * 60
    delta = torch.empty_like(y)
    gpu.connectedXentBackward(y, head.weights16, head.biases, labels, lse, None, 1.0, delta, head.bias_updates,
                              head.weight_updates, M, C, N)
    dy = delta.clone()
    dh = conv.backward(delta)
    # delta through relu is exact: 0 or itself
    assert torch.equal(delta, torch.where(y > 0, dy, torch.zeros_like(dy)))
    exact = P.connected_backward(h.view(M, C), conv.weights16, y, dy, P.RELU)
    tol = (C + 16) * 2 * U * (delta.double().abs() @ conv.weights16.double().abs())
    P.assert_within(dh, exact[1], tol + P.half_step(dh.dtype) * (exact[1].abs() + tol) + P.tiny(dh.dtype), "dh")
    tol = (M + 16) * 2 * U * (delta.double().abs().t() @ h.view(M, C).double().abs()) + 4 * U * exact[2].abs()
    P.assert_within(conv.weight_updates, exact[2], tol, "weight_updates")
    dx, bu, su = torch.empty_like(x), torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    gpu.gnActBackward(x, None if act == P.LOGISTIC else h, dh.view(B, S, C), dx, B, S, C, G, norm.scales, norm.biases,
                      norm.mean, norm.rstd, bu, su, act)
    assert torch.equal(norm.backward(dh.view(B, S, C)), dx)
    assert torch.equal(norm.bias_updates, bu) and torch.equal(norm.scale_updates, su)
    for layer in (conv, head):
        w, u = layer.weights.clone(), layer.weight_updates.clone()
        layer.update(0.1, 0.9, 0.0, M)
        change = 0.1 / M * u
        # the factor's, the product's and the sum's roundings, as in test_gpu_xent
        P.assert_within(layer.weights, w + change, 5 * U * (w.abs() + change.abs()), "weights")
        assert torch.equal(layer.weights16, layer.weights.bfloat16())
