"""The training-step operators' refusals: bad arguments come back as status codes or ValueError
before any device work, so they are checked without a GPU."""
import ctypes
import math

import pytest
import torch

P = ctypes.c_void_p(4096)   # an address that is never touched
NAN, INF = math.nan, math.inf


def _codes(pkg):
    return pkg._lib.lib(), pkg._lib.EC_OK, pkg._lib.EC_EINVAL, pkg._lib.EC_ERANGE, pkg._lib.EC_EALIGN


def test_embed_refusals(pkg):
    L, ok, inval, big, _ = _codes(pkg)

    def call(tokens=P, bytes_=8, n=4, table=P, kind=0, vocab=10, hidden=8, stride=8, start=0, scale=1.0, out=P):
        return L.ec_embed(tokens, bytes_, n, table, kind, vocab, hidden, stride, start, scale, out, None)

    assert call(n=0, tokens=None, out=None) == ok
    assert call(hidden=0, stride=0) == ok
    for bad in (dict(tokens=None), dict(bytes_=2), dict(table=None), dict(kind=3), dict(kind=-1), dict(stride=7),
                dict(scale=NAN), dict(scale=INF), dict(out=None)):
        assert call(**bad) == inval, bad
    assert call(n=1 << 31) == big
    assert call(hidden=(1 << 20) + 1, stride=1 << 21) == big


def test_embed_grad_refusals(pkg):
    L, ok, inval, big, align = _codes(pkg)
    need = L.ec_embed_grad_workspace(100, 10, 8)
    assert need > 0 and L.ec_embed_grad_workspace(1 << 31, 10, 8) == 0
    assert L.ec_embed_grad_workspace(0, 10, 8) == 0

    def call(tokens=P, bytes_=4, n=100, dout=P, kind=1, dstride=8, vocab=10, hidden=8, scale=1.0, grad=P,
             gkind=0, gstride=8, add=0, work=P, size=need):
        return L.ec_embed_grad(tokens, bytes_, n, dout, kind, dstride, vocab, hidden, 0, scale, grad, gkind,
                               gstride, add, work, size, None)

    assert call(vocab=0) == ok and call(hidden=0) == ok
    assert call(n=0, tokens=None, dout=None, add=1, work=None, size=0) == ok
    for bad in (dict(tokens=None), dict(bytes_=1), dict(dout=None), dict(kind=7), dict(dstride=7), dict(scale=NAN),
                dict(grad=None), dict(gkind=2), dict(gstride=7), dict(work=None), dict(size=need - 1)):
        assert call(**bad) == inval, bad
    assert call(work=ctypes.c_void_p(4100)) == align
    assert call(n=1 << 31) == big and call(vocab=1 << 31) == big


def test_token_logprobs_refusals(pkg):
    L, ok, inval, big, _ = _codes(pkg)

    def call(logits=P, kind=0, rows=4, vocab=50, stride=50, targets=P, scale=1.0, lp=P, lse=P, ent=None, top=0,
             tlp=None, tt=None):
        return L.ec_token_logprobs(logits, kind, rows, vocab, stride, targets, scale, lp, lse, ent, top, tlp, tt, None)

    assert call(rows=0, logits=None, targets=None, lp=None, lse=None) == ok
    for bad in (dict(logits=None), dict(kind=3), dict(stride=49), dict(targets=None), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=NAN), dict(scale=3e38), dict(lp=None), dict(lse=None), dict(top=-1), dict(top=3, tlp=P),
                dict(top=3, tt=P), dict(top=5, vocab=4, stride=4, tlp=P, tt=P)):
        assert call(**bad) == inval, bad
    assert call(top=17, tlp=P, tt=P) == big
    assert call(rows=1 << 31) == big and call(vocab=1 << 31, stride=1 << 31) == big


def test_token_logprobs_grad_refusals(pkg):
    L, ok, inval, big, _ = _codes(pkg)

    def call(logits=P, kind=0, rows=4, vocab=50, stride=50, targets=P, lse=P, dlp=P, ent=None, dent=None, scale=1.0,
             out=P, ostride=50):
        return L.ec_token_logprobs_grad(logits, kind, rows, vocab, stride, targets, lse, dlp, ent, dent, scale, out,
                                        ostride, None)

    assert call(rows=0) == ok and call(vocab=0, stride=0) == ok
    for bad in (dict(logits=None), dict(kind=3), dict(stride=49), dict(targets=None), dict(lse=None), dict(dlp=None),
                dict(ent=P), dict(dent=P), dict(scale=0.0), dict(out=None), dict(ostride=49)):
        assert call(**bad) == inval, bad
    assert call(rows=1 << 31) == big


def test_grad_list_refusals(pkg):
    L, _, inval, _, align = _codes(pkg)
    assert L.ec_grad_norm(None, 1, 1.0, 2, P, P, None) == inval
    for bad in ((P, 1, NAN, 2, P, P), (P, 1, 1.0, 1, P, P), (P, 1, 1.0, 2, None, P), (P, 1, 1.0, 2, P, None)):
        assert L.ec_grad_norm(*bad, None) == inval
    assert L.ec_grad_norm(P, 1, 1.0, 2, ctypes.c_void_p(4100), P, None) == align
    for most in (0.0, -1.0, NAN):
        assert L.ec_grad_clip(P, 1, 1.0, 2, most, None, P, P, None) == inval
    assert L.ec_grad_clip(P, 1, INF, 2, 1.0, None, P, P, None) == inval
    assert L.ec_grad_clip(P, 1, 1.0, 3, 1.0, None, P, P, None) == inval


def test_host_tensors_and_bad_factors_are_refused(pkg):
    table, tok = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    x, lse = torch.zeros(3, 50), torch.zeros(3)
    for call in (lambda: pkg.embed(tok, table), lambda: pkg.embed_grad(tok, torch.zeros(3, 8), 10),
                 lambda: pkg.token_logprobs(x, tok), lambda: pkg.token_logprobs_grad(x, tok, lse, lse),
                 lambda: pkg.grad_norm([table]), lambda: pkg.clip_grads([table], 1.0)):
        with pytest.raises(ValueError, match="device"):
            call()
    with pytest.raises(ValueError, match="finite"):
        pkg.embed(tok, table, scale=NAN)
    with pytest.raises(ValueError, match="positive"):
        pkg.token_logprobs(x, tok, scale=0.0)
    with pytest.raises(ValueError, match="dtype"):
        pkg.embed_grad(tok, torch.zeros(3, 8), 10, dtype=torch.float64)
    with pytest.raises(ValueError, match="float64|Double|double"):
        pkg.embed(tok, table.double())
