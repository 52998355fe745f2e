"""Arguments that the 16-bit entries refuse, on the CPU: the status comes back before a device is touched."""
from __future__ import annotations

import ctypes as C

import pytest

from darknet_zig_b200 import _lib

F32, BF16, F16 = 0, 1, 2
P = 1 << 20  # a stand-in for a device pointer; never dereferenced
INVALID, UNSUPPORTED = 1, 5


def status(name, *args):
    L = _lib.lib()
    fn = getattr(L, "dnb_" + name)
    assert len(fn.argtypes) == len(args), (name, len(fn.argtypes), len(args))
    st = fn(*args)
    if st:
        assert L.dnb_last_error_detail()
    return st


def gn_fwd(x=P, y=2 * P, dtype=BF16, B=2, S=4, Cn=8, G=2, sc=3 * P, bi=4 * P, eps=1e-5, mean=5 * P, rstd=6 * P, act=7,
           ws=None, wn=0):
    return status("gn_act_forward", x, y, dtype, B, S, Cn, G, sc, bi, eps, mean, rstd, act, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(S=-1), dict(Cn=0), dict(G=0), dict(G=3), dict(act=14),
    dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None), dict(sc=None), dict(bi=None), dict(mean=None),
    dict(rstd=None), dict(x=P + 1), dict(y=P + 16), dict(rstd=5 * P + 4), dict(mean=P), dict(B=1 << 40, S=1 << 40),
])
def test_gn_forward_refuses(built_lib, kw):
    assert gn_fwd(**kw) == INVALID


def test_gn_refuses_wide_groups_and_short_workspaces(built_lib):
    assert gn_fwd(Cn=8192, G=1) == UNSUPPORTED
    n = C.c_size_t(0)
    args = (BF16, 1, 1 << 20, 64, 1)
    assert status("gn_act_forward_workspace", P, 2 * P, *args, C.byref(n)) == 0 and n.value > 0
    big = dict(B=1, S=1 << 20, Cn=64, G=1, y=1 << 40, mean=1 << 41, rstd=1 << 42)
    assert gn_fwd(**big) == INVALID
    assert gn_fwd(**big, ws=1 << 43, wn=n.value - 1) == INVALID
    assert gn_fwd(**big, ws=(1 << 43) + 8, wn=n.value) == INVALID
    assert status("gn_act_forward_workspace", P, 2 * P, *args, None) == INVALID


def gn_bwd(x=P, y=None, d=2 * P, dx=3 * P, dtype=BF16, B=2, S=4, Cn=8, G=2, sc=4 * P, bi=5 * P, mean=6 * P, rstd=7 * P,
           bu=8 * P, su=9 * P, act=7, acc=0, ws=10 * P, wn=1 << 19):
    return status("gn_act_backward", x, y, d, dx, dtype, B, S, Cn, G, sc, bi, mean, rstd, bu, su, act, acc, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=9), dict(B=-1), dict(G=3), dict(act=-1), dict(acc=2), dict(acc=5), dict(x=None), dict(d=None),
    dict(dx=None), dict(sc=None), dict(bi=None), dict(mean=None), dict(rstd=None), dict(bu=None), dict(su=None),
    dict(dx=P), dict(y=3 * P), dict(dx=2 * P + 32), dict(su=8 * P + 4), dict(x=P + 1), dict(ws=None), dict(wn=1),
    dict(ws=10 * P + 4), dict(bu=3 * P),
])
def test_gn_backward_refuses(built_lib, kw):
    assert gn_bwd(**kw) == INVALID


def sgd(rows=4, cols=8, w=P, wu=2 * P, g=3 * P, ldg=8, w16=4 * P, ld16=8, dtype=BF16, batch=4):
    return status("sgd_momentum_mixed", rows, cols, w, wu, g, ldg, w16, ld16, dtype, 0.1, 0.9, 0.0, batch, None)


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(cols=-1), dict(dtype=F32), dict(batch=0), dict(w=None), dict(wu=None), dict(w16=None),
    dict(ldg=7), dict(ld16=7), dict(w=P + 2), dict(w16=4 * P + 1), dict(wu=P + 64), dict(w16=P), dict(g=2 * P),
    dict(g=4 * P, ldg=9), dict(rows=1 << 40, cols=1 << 40, ldg=1 << 40, ld16=1 << 40),
])
def test_sgd_refuses(built_lib, kw):
    assert sgd(**kw) == INVALID


def test_sgd_of_nothing(built_lib):
    assert sgd(rows=0) == 0 and sgd(cols=0, w=None) == 0


def conn_fwd(x=P, ldx=16, w=2 * P, ldw=16, b=3 * P, r=4 * P, ldr=8, y=5 * P, ldy=8, dtype=BF16, M=4, K=16, N=8, act=7,
             ws=None, wn=0):
    return status("connected_act_forward", x, ldx, w, ldw, b, r, ldr, y, ldy, dtype, M, K, N, act, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=F32), dict(dtype=7), dict(M=-1), dict(K=-1), dict(N=-1), dict(act=14), dict(x=None), dict(w=None),
    dict(y=None), dict(ldx=15), dict(ldw=15), dict(ldr=7), dict(ldy=7), dict(x=P + 1), dict(b=3 * P + 2), dict(y=P),
    dict(y=2 * P + 32), dict(y=3 * P), dict(y=4 * P, ldy=9), dict(y=4 * P + 16), dict(ldx=1 << 62),
    dict(M=100, x=P + 2, y=6 * P, ws=None), dict(M=100, ldx=17, y=6 * P, ws=7 * P, wn=10),
])
def test_connected_forward_refuses(built_lib, kw):
    assert conn_fwd(**kw) == INVALID


def test_connected_size_limits(built_lib):
    assert conn_fwd(M=1 << 31) == UNSUPPORTED
    assert conn_fwd(M=0, x=None, y=None) == 0 and conn_fwd(N=0, w=None) == 0


def conn_bwd(x=P, ldx=16, w=2 * P, ldw=16, y=3 * P, ldy=8, d=4 * P, ldd=8, dz=5 * P, lddz=8, dx=6 * P, lddx=16, bu=7 * P,
             wu=8 * P, lddw=16, ut=F32, dtype=BF16, M=4, K=16, N=8, act=7, acc=0, ws=9 * P, wn=1 << 19):
    return status("connected_act_backward", x, ldx, w, ldw, y, ldy, d, ldd, dz, lddz, dx, lddx, bu, wu, lddw, ut, dtype,
                  M, K, N, act, acc, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=F32), dict(ut=F16), dict(ut=9), dict(M=-1), dict(act=99), dict(acc=4), dict(x=None), dict(w=None),
    dict(y=None), dict(d=None), dict(dz=None), dict(ldx=3), dict(ldd=7), dict(lddz=7), dict(lddx=15), dict(lddw=15),
    dict(wu=8 * P + 2), dict(bu=7 * P + 1), dict(dx=P), dict(dx=4 * P), dict(wu=2 * P), dict(dz=4 * P, lddz=9),
    dict(dz=3 * P), dict(bu=8 * P), dict(dx=5 * P), dict(ws=None), dict(wn=16), dict(ws=9 * P + 8),
])
def test_connected_backward_refuses(built_lib, kw):
    assert conn_bwd(**kw) == INVALID


def xent_fwd(x=P, ldx=16, w=2 * P, ldw=16, b=3 * P, lab=4 * P, loss=5 * P, lse=6 * P, dtype=BF16, M=4, K=16, N=8,
             ws=7 * P, wn=1 << 19):
    return status("connected_xent_forward", x, ldx, w, ldw, b, lab, loss, lse, dtype, M, K, N, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=F32), dict(M=-1), dict(K=0), dict(N=0), dict(x=None), dict(w=None), dict(lab=None), dict(loss=None),
    dict(lse=None), dict(ldx=15), dict(ldw=1), dict(x=P + 1), dict(lab=4 * P + 2), dict(loss=5 * P + 1),
    dict(lse=5 * P), dict(loss=P), dict(lse=4 * P), dict(ws=None), dict(wn=8), dict(ws=7 * P + 4),
])
def test_xent_forward_refuses(built_lib, kw):
    assert xent_fwd(**kw) == INVALID


def xent_bwd(x=P, ldx=16, w=2 * P, ldw=16, b=3 * P, lab=4 * P, lse=5 * P, rs=6 * P, dx=7 * P, lddx=16, bu=8 * P,
             wu=9 * P, lddw=16, ut=F32, dtype=BF16, M=4, K=16, N=8, acc=0, ws=10 * P, wn=1 << 19):
    return status("connected_xent_backward", x, ldx, w, ldw, b, lab, lse, rs, 1.0, dx, lddx, bu, wu, lddw, ut, dtype, M,
                  K, N, acc, ws, wn, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=F32), dict(ut=F16), dict(M=-1), dict(K=0), dict(N=0), dict(acc=8), dict(x=None), dict(w=None),
    dict(lab=None), dict(lse=None), dict(ldx=15), dict(ldw=15), dict(lddx=15), dict(lddw=15), dict(rs=6 * P + 2),
    dict(dx=P), dict(wu=2 * P), dict(bu=3 * P), dict(wu=7 * P), dict(bu=5 * P), dict(ws=None), dict(wn=64),
    dict(ws=10 * P + 8),
])
def test_xent_backward_refuses(built_lib, kw):
    assert xent_bwd(**kw) == INVALID
