"""Refusals of the block operators' C entry points and of host tensors, without a GPU: every call returns before any
device work, so the addresses are never touched."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4104)
NAN, INF = float("nan"), float("inf")


def _codes(pkg):
    return pkg._lib.lib(), pkg._lib.EC_OK, pkg._lib.EC_EINVAL, pkg._lib.EC_ERANGE, pkg._lib.EC_EALIGN


def test_gated_ff_refusals(pkg):
    L, ok, inval, big, align = _codes(pkg)

    def call(x=P, xs=32, g=P, gs=32, u=P, us=32, kind=1, n=4, width=32, inner=48, act=0, h=P, hs=48, work=None, have=0):
        return L.ec_gated_ff(x, xs, g, gs, u, us, kind, n, width, inner, act, h, hs, work, have, None)

    assert call(n=0) == ok and call(n=0, x=None, h=None) == ok
    for bad in (dict(x=None), dict(g=None), dict(u=None), dict(h=None), dict(kind=3), dict(kind=-1), dict(act=3), dict(act=-1),
                dict(xs=31), dict(gs=31), dict(us=31), dict(hs=47), dict(width=0, xs=0), dict(inner=0),
                dict(n=99, x=ctypes.c_void_p(4098)), dict(n=99, xs=33), dict(n=99, width=31)):   # the last need a workspace
        assert call(**bad) == inval, bad
    for bad in (dict(n=1 << 31), dict(width=(1 << 19) + 1, xs=1 << 20, gs=1 << 20, us=1 << 20),
                dict(inner=(1 << 19) + 1, hs=1 << 20), dict(n=(1 << 31) - 1, inner=1 << 19, hs=1 << 20),
                dict(n=1 << 30), dict(inner=1 << 19, width=1 << 19, xs=1 << 19, gs=1 << 19, us=1 << 19, hs=1 << 19)):
        assert call(**bad) == big, bad
    need = L.ec_gated_ff_workspace(P, 31, P, 32, P, 32, 1, 99, 31, 48, 0)
    assert need >= 99 * 64 + 2 * 48 * 64 and L.ec_gated_ff_workspace(P, 32, P, 32, P, 32, 1, 99, 32, 48, 0) == 0
    assert L.ec_gated_ff_workspace(P, 31, P, 31, P, 31, 1, 4, 31, 48, 0) == 0   # few rows are read as they are
    assert call(n=99, width=31, xs=31, work=P, have=need - 1) == inval
    # weights of different strides are copied, both
    assert L.ec_gated_ff_workspace(P, 32, P, 32, P, 40, 1, 99, 32, 48, 0) >= 2 * 48 * 64 and call(n=99, us=40) == inval
    assert call(n=99, width=31, xs=31, work=ODD, have=need) == align
    assert L.ec_gated_ff_workspace(P, 32, P, 32, P, 32, 7, 4, 32, 48, 0) == 0


def test_gated_ff_grad_refusals(pkg):
    L, ok, inval, big, align = _codes(pkg)

    def call(dh=P, dhs=48, x=P, xs=32, g=P, gs=32, u=P, us=32, kind=1, n=4, width=32, inner=48, act=0, dx=P, dxs=32, dg=P,
             dgs=32, du=P, dus=32, out=1, acc=0, work=P, have=1 << 20):
        return L.ec_gated_ff_grad(dh, dhs, x, xs, g, gs, u, us, kind, n, width, inner, act, dx, dxs, dg, dgs, du, dus, out, acc,
                                  work, have, None)

    assert call(n=0, acc=1) == ok and call(n=0, dg=None, du=None) == ok
    need = L.ec_gated_ff_workspace(P, 32, P, 32, P, 32, 1, 4, 32, 48, 1)
    assert need >= 4 * 96 * 2 * 2
    for bad in (dict(dh=None), dict(x=None), dict(dhs=47), dict(dxs=31), dict(dgs=31), dict(dus=31), dict(dg=None),
                dict(du=None), dict(dx=None, dg=None, du=None), dict(out=2), dict(out=5), dict(act=9), dict(have=need - 1),
                dict(work=None)):
        assert call(**bad) == inval, bad
    assert call(work=ODD) == align and call(n=1 << 31) == big


def test_orthogonalize_refusals(pkg):
    L, ok, inval, big, align = _codes(pkg)
    abc = (ctypes.c_float * 3)(3.4445, -4.775, 2.0315)

    def call(x=P, kind=1, batch=2, rows=130, cols=150, xs=150, xm=19500, steps=5, coef=abc, eps=1e-7, scale=1.0, base=None,
             bs=0, bm=0, keep=1.0, out=P, okind=0, os=150, om=19500, work=P, have=1 << 28):
        return L.ec_orthogonalize(x, kind, batch, rows, cols, xs, xm, steps, coef, eps, scale, base, bs, bm, keep, out, okind,
                                  os, om, work, have, None)

    assert call(batch=0) == ok and call(batch=0, x=None, out=None, work=None) == ok
    need = L.ec_orthogonalize_workspace(2, 130, 150)
    assert need >= 2 * 4 * (2 * 130 * 152 + 2 * 130 * 136)
    assert L.ec_orthogonalize_workspace(2, 128, 128) == 0   # small ones need none
    for bad in (dict(x=None), dict(out=None), dict(kind=4), dict(okind=-1), dict(rows=0), dict(cols=0), dict(xs=149), dict(os=149),
                dict(base=P, bs=149), dict(eps=0.0), dict(eps=NAN), dict(eps=INF), dict(scale=INF), dict(keep=NAN), dict(coef=None),
                dict(coef=(ctypes.c_float * 3)(1, NAN, 0)), dict(coef=(ctypes.c_float * 3)(1, 1025, 0)), dict(work=None),
                dict(have=need - 1)):
        assert call(**bad) == inval, bad
    for bad in (dict(rows=65537), dict(cols=65537, xs=65537, os=65537), dict(batch=65537), dict(steps=0), dict(steps=65)):
        assert call(**bad) == big, bad
    assert call(work=ODD) == align
    assert L.ec_orthogonalize_workspace(0, 3, 3) == L.ec_orthogonalize_workspace(1, 0, 3) == 0


def test_residual_norm_refusals(pkg):
    L, ok, inval, big, _ = _codes(pkg)

    def call(r=P, rs=64, b=P, bs=64, kind=1, n=6, width=64, gate=P, gates=3, scale=1.0, bw=P, w=P, eps=1e-6, total=P, ts=64,
             normed=P):
        return L.ec_residual_norm(r, rs, b, bs, kind, n, width, gate, gates, scale, bw, w, eps, total, ts, normed, None, None, None)

    assert call(n=0) == ok and call(n=0, r=None, total=None, normed=None) == ok
    for bad in (dict(r=None), dict(rs=63), dict(bs=63), dict(ts=63), dict(kind=3), dict(width=0), dict(gates=0), dict(gates=4),
                dict(scale=NAN), dict(eps=-1.0), dict(eps=INF), dict(total=None), dict(normed=None), dict(b=None),
                dict(b=None, gate=None), dict(b=None, gate=None, bw=None, w=None)):
        assert call(**bad) == inval, bad
    assert call(n=1 << 31, gates=1) == big and call(width=16385, rs=16385, bs=16385, ts=16385) == big


def test_residual_norm_grad_refusals(pkg):
    L, _, inval, big, align = _codes(pkg)

    def call(ds=P, dss=64, dn=P, dns=64, s=P, ss=64, b=P, bs=64, kind=1, n=6, width=64, rstd=P, brstd=P, gate=P, gates=3, scale=1.0,
             bw=P, w=P, dr=P, db=P, dg=P, dbw=P, dw=P, work=P, have=1 << 24):
        return L.ec_residual_norm_grad(ds, dss, dn, dns, s, ss, b, bs, kind, n, width, rstd, brstd, gate, gates, scale, bw, w, dr,
                                       db, dg, dbw, dw, work, have, None)

    need = L.ec_residual_norm_grad_workspace(6, 64, 3)
    for bad in (dict(dss=63), dict(dns=63), dict(ss=63), dict(bs=63), dict(kind=5), dict(width=0), dict(gates=5), dict(gates=0),
                dict(rstd=None), dict(brstd=None), dict(dn=None), dict(s=None), dict(b=None), dict(dr=None), dict(db=None),
                dict(dg=None), dict(gate=None), dict(bw=None), dict(w=None), dict(ds=None, w=None, dw=None), dict(scale=INF),
                dict(work=None), dict(have=need - 1)):
        assert call(**bad) == inval, bad
    assert call(work=ODD) == align and call(n=1 << 31, gates=1) == big and call(n=0, gates=1 << 40) == big
    assert L.ec_residual_norm_grad_workspace(6, 64, 4) == 0


def test_host_tensors_and_bad_arguments_are_refused(pkg):
    x, w, v = torch.zeros(3, 8), torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: pkg.gated_ff(x, w, w), lambda: pkg.gated_ff_grad(torch.zeros(3, 4), x, w, w), lambda: pkg.orthogonalize(x),
                 lambda: pkg.residual_norm(x, x, weight=v), lambda: pkg.residual_norm_grad(x, None, x, x)):
        with pytest.raises(ValueError, match="device"):
            call()
    for call, what in ((lambda: pkg.gated_ff(x, w, w, activation="relu6"), "activation"),
                       (lambda: pkg.orthogonalize(x, eps=-1.0), "eps"), (lambda: pkg.orthogonalize(x, keep=INF), "finite"),
                       (lambda: pkg.residual_norm(x, x, scale=NAN), "finite"),
                       (lambda: pkg.gated_ff_grad(x, x, w, w, dtype=torch.int8), "dtype")):
        with pytest.raises(ValueError, match=what):
            call()
