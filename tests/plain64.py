"""Plain fp64 forms of the 16-bit entries (torch, any device), with darknet's activation numbering and
sign of deltas. The GPU tests compare the kernels with these; test_plain64_cpu.py compares the backward
formulas here with differences of the forward ones."""
from __future__ import annotations

import torch

LOGISTIC, RELU, LINEAR, TANH, LEAKY = 0, 1, 3, 5, 7
ACTS = {"logistic": LOGISTIC, "relu": RELU, "linear": LINEAR, "tanh": TANH, "leaky": LEAKY}
U = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype) -> float:
    """Half a step of the type, relative: how far one rounding to it may move a value."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half of the smallest subnormal: the absolute floor of a rounding to the type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def act(z, a):
    if a == LOGISTIC:
        return torch.sigmoid(z)
    if a == RELU:
        return z.clamp(min=0)
    if a == TANH:
        return torch.tanh(z)
    if a == LEAKY:
        return torch.where(z > 0, z, 0.1 * z)
    return z


def act_gradient(y, a):
    if a == LOGISTIC:
        return (1 - y) * y
    if a == RELU:
        return (y > 0).to(y.dtype)
    if a == TANH:
        return 1 - y * y
    if a == LEAKY:
        return torch.where(y > 0, torch.ones_like(y), torch.full_like(y, 0.1))
    return torch.ones_like(y)


def gn_stats(x, groups, eps):
    """mean and rstd [batch, groups] of x [batch, spatial, filters]."""
    B, S, C = x.shape
    v = x.double().reshape(B, S, groups, C // groups)
    mean = v.mean(dim=(1, 3))
    var = ((v - mean[:, None, :, None]) ** 2).mean(dim=(1, 3))
    return mean, 1 / torch.sqrt(var + eps)


def _wide(a, per):
    """[batch, groups] -> [batch, 1, filters]"""
    return a.double().repeat_interleave(per, dim=1)[:, None, :]


def gn_forward(x, groups, scales, biases, eps, a):
    mean, rstd = gn_stats(x, groups, eps)
    per = x.shape[2] // groups
    xh = (x.double() - _wide(mean, per)) * _wide(rstd, per)
    return act(xh * scales.double() + biases.double(), a), mean, rstd


def gn_backward(x, y, delta, groups, scales, biases, mean, rstd, a):
    """dx, bias_updates, scale_updates and the pieces a tolerance needs."""
    B, S, C = x.shape
    per = C // groups
    xh = (x.double() - _wide(mean, per)) * _wide(rstd, per)
    out = act(xh * scales.double() + biases.double(), a) if y is None else y.double()
    d = delta.double() * act_gradient(out, a)
    t = d * scales.double()
    gmean = lambda v: v.reshape(B, S, groups, per).mean(dim=(1, 3))  # noqa: E731
    m0, m1 = _wide(gmean(t), per), _wide(gmean(t * xh), per)
    dx = _wide(rstd, per) * (t - m0 - xh * m1)
    return dx, d.sum(dim=(0, 1)), (d * xh).sum(dim=(0, 1)), dict(
        xh=xh, d=d, t=t, m0=m0, m1=m1, a0=_wide(gmean(t.abs()), per), a1=_wide(gmean((t * xh).abs()), per),
        rstd=_wide(rstd, per), mean=_wide(mean, per))


def connected_forward(x, w, biases, residual, a):
    z = x.double() @ w.double().t()
    if biases is not None:
        z = z + biases.double()
    if residual is not None:
        z = z + residual.double()
    return act(z, a)


def connected_backward(x, w, y, delta, a):
    """dz, dx, weight_updates, bias_updates; the products take dz unrounded."""
    dz = delta.double() if a == LINEAR else delta.double() * act_gradient(y.double(), a)
    return dz, dz @ w.double(), dz.t() @ x.double(), dz.sum(dim=0)


def xent_forward(x, w, biases, labels):
    z = x.double() @ w.double().t()
    if biases is not None:
        z = z + biases.double()
    lse = torch.logsumexp(z, dim=1)
    valid = (labels >= 0) & (labels < w.shape[0])
    at = z.gather(1, labels.long().clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    return torch.where(valid, lse - at, torch.zeros_like(lse)), torch.where(valid, lse, torch.zeros_like(lse))


def xent_deltas(x, w, biases, labels, row_scales, scale):
    """d [batch, classes], 0 in padding rows (whose x may hold anything)."""
    valid = (labels >= 0) & (labels < w.shape[0])
    x = torch.where(valid[:, None], x.double(), torch.zeros_like(x, dtype=torch.float64))
    z = x @ w.double().t()
    if biases is not None:
        z = z + biases.double()
    d = -torch.softmax(z, dim=1)
    rows = torch.arange(x.shape[0], device=x.device)
    d[rows, labels.long().clamp(0, w.shape[0] - 1)] += 1
    d = d * scale
    if row_scales is not None:
        d = d * row_scales.double()[:, None]
    return torch.where(valid[:, None], d, torch.zeros_like(d)), x


def xent_backward(x, w, biases, labels, row_scales, scale):
    """dx, weight_updates, bias_updates, d."""
    d, x = xent_deltas(x, w, biases, labels, row_scales, scale)
    return d @ w.double(), d.t() @ x, d.sum(dim=0), d


def assert_within(got, want, tol, name):
    """|got - want| <= tol elementwise; not-a-numbers and infinities in the same places."""
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand_as(want)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{name}: infinities"
    err = (got - want).abs()
    bad = fine & ~(err <= tol)
    if bad.any():
        i = int(torch.where(fine, err / tol.clamp(min=1e-300), torch.zeros_like(err)).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got "
                             f"{got.flatten()[i].item()!r} want {want.flatten()[i].item()!r} tol "
                             f"{tol.flatten()[i].item()!r}")
