"""The training-step operators on the GPU against plain 64-bit implementations: sizes from one element on,
odd and strided rows, every type, masks that leave a row empty, values of the type's ends, repeated and
out-of-slice tokens.

Bounds.  u is half the spacing of the result's type relative to it (eps / 2) and `tiny` half its
smallest step; e = 2^-24 is that of the fp32 arithmetic.  A sum of n terms in fp32 is off by at most n e times
the sum of magnitudes, whatever its order.  exp2 and log2 of the hardware are taken as 2 e off."""
import importlib.util
import math
import os
import zlib

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}
types = pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)


def gen(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def check(got, want, bound, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    sane = want.isfinite()
    assert torch.equal(got[~sane & ~want.isnan()], want[~sane & ~want.isnan()]), f"{what}: infinities"
    bound = torch.as_tensor(bound, dtype=torch.float64).expand_as(want)
    off = (got - want).abs()[sane] - bound[sane]
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"{what}: {int((off > 0).sum())} of {off.numel()} over the bound, by {float(off.max()):.3g}"


def rounded(want, dtype, more=0.0):
    """Bound of a result rounded to dtype whose fp32 value is off by `more`."""
    return want.abs() * UNIT[dtype] * 1.01 + TINY[dtype] + more * 1.01


# --------------------------------------------------------------- embedding --

HIDDENS = [1, 3, 4, 7, 8, 9, 31, 64, 255, 513, 2048, 2049]


@types
@pytest.mark.parametrize("hidden", HIDDENS)
def test_embed(pkg, dev, dtype, hidden):
    g = gen("embed", hidden)
    vocab, n = 97, 61
    table = torch.randn(vocab, hidden, generator=g).to(dtype)
    tok = torch.randint(-40, 200, (n,), generator=g)
    tok[:4] = torch.tensor([10, 106, 9, 107])        # the slice's ends and their neighbours
    want = torch.zeros(n, hidden, dtype=torch.float64)
    here = (tok >= 10) & (tok < 107)
    want[here] = table[tok[here] - 10].double() * 1.7
    for ids in (torch.int64, torch.int32):
        got = pkg.embed(tok.to(ids).to(dev), table.to(dev), scale=1.7, vocab_start=10)
        assert got.dtype == dtype and got.shape == (n, hidden)
        check(got, want, rounded(want, dtype, want.abs() * 2 * E), "embed")
        assert not bool(got.cpu()[~here].any())


@types
def test_embed_shapes_strides_and_offsets(pkg, dev, dtype):
    g = gen("embed views")
    wide = torch.randn(50, 300, generator=g).to(dtype).to(dev)
    tok = torch.randint(0, 50, (3, 5, 2), generator=g).to(dev)
    for lo, hi in ((0, 300), (1, 34), (7, 264), (3, 10)):
        table = wide[:, lo:hi]
        got = pkg.embed(tok, table)
        assert torch.equal(got, table[tok])
    # an output that is a view at an odd element of a guarded buffer
    buf = torch.full((4 * 33 + 5,), 7.0, dtype=dtype, device=dev)
    pkg.embed(tok[0, :2].reshape(-1)[:4], wide[:, :33], out=buf[3:3 + 4 * 33].view(4, 33))
    assert torch.equal(buf[3:-2].view(4, 33), wide[:, :33][tok[0, :2].reshape(-1)[:4]])
    assert bool((buf[:3] == 7).all()) and bool((buf[-2:] == 7).all())
    assert pkg.embed(tok[:0], wide).shape == (0, 5, 2, 300)
    one = pkg.embed(tok[0, 0, :1], wide[:1].expand(1, 300), vocab_start=int(tok[0, 0, 0]))
    assert torch.equal(one, wide[:1])
    none = pkg.embed(tok, wide[:0])
    assert none.shape == (3, 5, 2, 300) and not bool(none.any())


def test_embed_any_token_value(pkg, dev):
    """Starts and tokens at the ends of 64 bits: a difference that wraps is no row."""
    table = torch.arange(1.0, 5.0, device=dev).view(4, 1)
    lo, hi = -(1 << 63), (1 << 63) - 1
    tok = torch.tensor([lo, lo + 1, -1, 0, 3, 4, hi - 1, hi], device=dev)
    assert pkg.embed(tok, table)[:, 0].tolist() == [0, 0, 0, 1, 4, 0, 0, 0]
    assert pkg.embed(tok, table, vocab_start=lo)[:, 0].tolist() == [1, 2, 0, 0, 0, 0, 0, 0]
    assert pkg.embed(tok, table, vocab_start=hi - 1)[:, 0].tolist() == [0, 0, 0, 0, 0, 0, 1, 2]


def egrad_want(tok, dout, vocab, start, scale):
    here = (tok >= start) & (tok < start + vocab)
    rows = tok[here] - start
    want = torch.zeros(vocab, dout.shape[-1], dtype=torch.float64).index_add_(0, rows, dout[here].double())
    size = torch.zeros_like(want).index_add_(0, rows, dout[here].double().abs())
    count = torch.zeros(vocab, 1, dtype=torch.float64).index_add_(0, rows, torch.ones(len(rows), 1, dtype=torch.float64))
    return want * scale, (count + 2) * E * size * abs(scale), count


@types
@pytest.mark.parametrize("n,hidden,vocab", [(1, 5, 3), (2, 8, 1), (31, 64, 40), (32, 9, 7), (33, 513, 200), (64, 16, 2),
                                            (500, 33, 60), (4096, 8, 5000), (4097, 40, 300), (9000, 17, 1 << 21)])
def test_embed_grad(pkg, dev, dtype, n, hidden, vocab):
    g = gen("egrad", n, hidden)
    dout = torch.randn(n, hidden, generator=g).to(dtype)
    tok = torch.randint(-2, vocab + 3, (n,), generator=g)
    want, more, _ = egrad_want(tok, dout, vocab, 0, 0.3)
    for out in {torch.float32, dtype}:
        got = pkg.embed_grad(tok.to(dev), dout.to(dev), vocab, scale=0.3, dtype=out)
        assert got.dtype == out
        check(got, want, rounded(want, out, more), f"egrad {out}")


@pytest.mark.parametrize("n,vocab,hidden", [(8192, 3000, 24), (8193, 3000, 24), (10_000, 70_001, 40), (16_385, 262_144, 8),
                                            (33_000, 262_145, 8), (40_000, 1000, 1)])
def test_embed_grad_over_its_rules(pkg, dev, n, vocab, hidden):
    """Both sides of the sizes where the sort, its digits, the tiles and the zeros' bits change."""
    g = gen("rules", n)
    dout = torch.randn(n, hidden, generator=g).bfloat16()
    tok = (torch.rand(n, generator=g) ** 4 * (vocab + 9)).long()
    tok[::97] = vocab - 1
    want, more, count = egrad_want(tok, dout, vocab, 0, 1.0)
    buf = torch.full((vocab * hidden + 16,), 7.0, device=dev)
    out = buf[8:-8].view(vocab, hidden)
    got = pkg.embed_grad(tok.to(dev), dout.to(dev), vocab, out=out)
    check(got, want, rounded(want, torch.float32, more), "rules")
    assert not bool(got.cpu()[count[:, 0] == 0].any())
    assert bool((buf[:8] == 7).all()) and bool((buf[-8:] == 7).all())
    pkg.embed_grad(tok.to(dev), dout.to(dev), vocab, out=out, accumulate=True)
    check(out, want * 2, rounded(want * 2, torch.float32, more * 2 + want.abs() * 2 * E), "twice")


@pytest.mark.parametrize("n", [5, 9000])
@pytest.mark.parametrize("hidden,pad", [(1, 0), (3, 0), (7, 0), (8, 0), (9, 0), (33, 0), (250, 0), (511, 0), (513, 0), (33, 4),
                                        (300, 1), (700, 5)])
@types
def test_embed_grad_zeros_between_rows(pkg, dev, dtype, hidden, pad, n):
    """Rows of zeros next to rows that occur, narrow ones that share 16 bytes and lines, dense and strided, into
    a gradient that held something else, at an odd element."""
    g = gen("zeros", hidden, pad, n)
    vocab = 2600
    dout = torch.randn(n, hidden, generator=g).to(dtype)
    tok = torch.randint(0, 900, (n,), generator=g) * 3 % vocab
    tok[0], tok[1] = 0, vocab - 1
    buf = torch.full((vocab * (hidden + pad) + 9,), 7.0, dtype=dtype, device=dev)
    out = buf[3:3 + vocab * (hidden + pad)].view(vocab, hidden + pad)[:, :hidden]
    got = pkg.embed_grad(tok.to(dev), dout.to(dev), vocab, out=out)
    want, more, count = egrad_want(tok, dout, vocab, 0, 1.0)
    check(got, want, rounded(want, dtype, more), "zeros between")
    assert not bool(got.cpu()[count[:, 0] == 0].any())
    rest = buf.cpu()
    inside = torch.zeros(rest.numel(), dtype=torch.bool)
    inside[3:3 + vocab * (hidden + pad)].view(vocab, hidden + pad)[:, :hidden] = True
    assert bool((rest[~inside] == 7).all())


@pytest.mark.parametrize("how", ["one token", "two tokens", "none inside", "a tenth"])
def test_embed_grad_of_repeated_tokens(pkg, dev, how):
    """Runs over many tiles, their ends anywhere, and slices that nobody asks for."""
    n, hidden, vocab = 20_011, 72, 500
    g = gen("repeat", how)
    dout = torch.randn(n, hidden, generator=g)
    tok = torch.randint(0, vocab, (n,), generator=g)
    if how == "one token":
        tok[:] = 123
    elif how == "two tokens":
        tok = torch.where(torch.arange(n) % 3 == 0, 499, 0)
    elif how == "none inside":
        tok += 500
    else:
        tok[torch.rand(n, generator=g) < 0.1] = 77
    want, more, count = egrad_want(tok, dout, vocab, 0, 1.0)
    got = pkg.embed_grad(tok.int().to(dev), dout.to(dev), vocab)
    check(got, want, rounded(want, torch.float32, more), how)
    again = pkg.embed_grad(tok.int().to(dev), dout.to(dev), vocab)
    assert torch.equal(got, again)
    assert not bool(got.cpu()[count[:, 0] == 0].any())


@types
def test_embed_grad_accumulates_into_views(pkg, dev, dtype):
    """Strided dout and gradient, odd starts; rows of tokens that do not occur keep their bits."""
    g = gen("acc")
    n, vocab, hidden = 300, 50, 37
    wide = torch.randn(n, 64, generator=g).to(dtype).to(dev)
    dout = wide[:, 5:5 + hidden]
    tok = torch.randint(0, vocab, (n,), generator=g)
    tok[tok == 7] = 8
    base = torch.full((vocab, 96), 3.25, device=dev)
    base[7, 20] = math.nan
    grad = base[:, 11:11 + hidden]
    before = grad.clone()
    got = pkg.embed_grad(tok.to(dev), dout, vocab, scale=0.5, out=grad, accumulate=True)
    assert got.data_ptr() == grad.data_ptr()
    want, more, _ = egrad_want(tok, dout.cpu(), vocab, 0, 0.5)
    want += before.double().cpu()
    check(grad, want, rounded(want, torch.float32, more + want.abs() * E), "accumulate")
    assert bool((base[:, :11] == 3.25).all()) and bool((base[:, 11 + hidden:] == 3.25).all())
    pkg.embed_grad(tok.to(dev), dout, vocab, scale=0.5, out=grad)     # written, not added
    want, more, _ = egrad_want(tok, dout.cpu(), vocab, 0, 0.5)
    check(grad, want, rounded(want, torch.float32, more), "written")
    assert bool((base[:, :11] == 3.25).all()) and bool((base[:, 11 + hidden:] == 3.25).all())


def test_embed_grad_of_nothing(pkg, dev):
    empty = torch.zeros(0, dtype=torch.int64, device=dev)
    got = pkg.embed_grad(empty, torch.zeros(0, 12, device=dev), 9)
    assert got.shape == (9, 12) and not bool(got.any())
    keep = torch.ones(9, 12, device=dev)
    pkg.embed_grad(empty, torch.zeros(0, 12, device=dev), 9, out=keep, accumulate=True)
    assert bool((keep == 1).all())
    assert pkg.embed_grad(empty, torch.zeros(0, 12, device=dev), 0).shape == (0, 12)


def test_embed_differences(pkg, dev):
    """The lookup is linear, so the difference quotient of <dout, embed(table)> is the gradient; through
    autograd, in the table's type."""
    g = gen("embed diff")
    vocab, hidden, n = 6, 5, 40
    table = torch.randn(vocab, hidden, generator=g).to(dev).requires_grad_()
    tok = torch.randint(0, vocab + 2, (n,), generator=g).to(dev)
    dout = torch.randn(n, hidden, generator=g).to(dev)
    pkg.embed(tok, table, scale=1.5).backward(dout)
    for v in range(vocab):
        for c in range(hidden):
            ends = []
            for sign in (1, -1):
                t = table.detach().clone()
                t[v, c] = 2.0 * sign
                ends.append(float((pkg.embed(tok, t, scale=1.5).double() * dout.double()).sum()))
            assert abs((ends[0] - ends[1]) / 4 - float(table.grad[v, c])) <= (n + 4) * E * 1.5 * n * 5
    assert pkg.embed(tok, table.detach()).requires_grad is False
    # a broadcast gradient: every row the same memory
    table.grad = None
    pkg.embed(tok, table).sum().backward()
    counts = torch.bincount(tok.cpu(), minlength=vocab)[:vocab].float()
    assert torch.equal(table.grad.cpu(), counts[:, None].expand(vocab, hidden))


# ------------------------------------------------------- log probabilities --

def logp_want(x, target, scale):
    z = x.double() * scale
    lse = z.logsumexp(1)
    p = (z - lse[:, None]).exp()
    ent = -torch.where(p > 0, p * (z - lse[:, None]), 0.0).sum(1)
    ok = (target >= 0) & (target < x.shape[1])
    lp = torch.where(ok, z.gather(1, torch.where(ok, target, 0)[:, None])[:, 0] - lse, 0.0)
    return z, lse, lp, ent, p


def logp_bounds(x, scale, lp):
    """(bound of lse, of log probabilities, of entropies) for rows whose finite logits are at most R from 0: a lane
    adds a 256th of the row, then 20 partial sums; an exponent is off by 2 e of its size."""
    finite = torch.where(x.double().isfinite(), x.double() * scale, 0.0)
    R = finite.abs().amax(1)
    top = finite.amax(1)
    adds = x.shape[1] / 256 + 8 + 20
    s = (adds + 4 + 4 * (R + 1)) * E          # relative error of the sum of exponentials
    return s + 4 * E * (R + 12), s + 4 * E * (lp.abs().nan_to_num(posinf=0, neginf=0) + 12 + (R - top).abs() * 0), \
        (s * 4 + 16 * E) * (R + 12)


@types
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (2, 8), (4, 63), (9, 257), (3, 2047), (3, 2049), (2, 8192),
                                        (7, 16411), (2, 50304), (1, 151_937)])
def test_token_logprobs(pkg, dev, dtype, rows, vocab):
    g = gen("logp", rows, vocab)
    x = (torch.randn(rows, vocab, generator=g) * 4).to(dtype)
    x[torch.rand(rows, vocab, generator=g) < 0.1] = -math.inf
    x[:, 0] = 1.0
    target = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        target[0], target[1] = -100, vocab
    top = min(vocab, 16)
    z, lse, lp, ent, _ = logp_want(x, target, 0.8)
    b_lse, b_lp, b_ent = logp_bounds(x, 0.8, lp)
    r = pkg.token_logprobs(x.to(dev), target.to(dev), scale=0.8, entropy=True, top=top)
    check(r.lse, lse, b_lse, "lse")
    check(r.logprobs, lp, b_lp, "logprobs")
    check(r.entropy, ent, b_ent, "entropy")
    order = x.double().argsort(dim=1, descending=True, stable=True)[:, :top]
    assert torch.equal(r.top_tokens.cpu(), order)
    want = z.gather(1, order) - lse[:, None]
    check(r.top_logprobs, want, logp_bounds(x, 0.8, lp)[1][:, None] + 4 * E * want.abs().nan_to_num(posinf=0), "top")
    bare = pkg.token_logprobs(x.to(dev), target.to(dev), scale=0.8)
    assert bare.entropy is None and bare.top_tokens is None
    assert torch.equal(bare.logprobs, r.logprobs) and torch.equal(bare.lse, r.lse)
    one = pkg.token_logprobs(x.to(dev), target.to(dev), scale=0.8, top=1)
    assert torch.equal(one.top_tokens, r.top_tokens[:, :1])
    assert torch.equal(one.top_logprobs, r.top_logprobs[:, :1])


@types
def test_token_logprobs_ties_go_to_the_lowest_index(pkg, dev, dtype):
    vocab = 50_000
    rows = torch.zeros(5, vocab)
    rows[1] = torch.arange(vocab) % 7                          # the largest value thousands of times
    rows[2, ::2] = -0.0                                        # both zeros are one value
    rows[3] = -math.inf
    rows[3, [49_999, 3, 20_000]] = torch.tensor([1.0, 1.0, 2.0])   # fewer than `top` are unmasked
    rows[4] = -torch.arange(vocab) / 1000
    rows[4, 100:] = -math.inf
    x = rows.to(dtype)
    r = pkg.token_logprobs(x.to(dev), torch.zeros(5, dtype=torch.int64, device=dev), top=16)
    order = x.double().argsort(dim=1, descending=True, stable=True)[:, :16]
    assert torch.equal(r.top_tokens.cpu(), order)


@types
def test_token_logprobs_top_where_the_candidates_overflow(pkg, dev, dtype):
    """Large logits at one place of every stretch that the workgroup's lanes share, and ascending rows."""
    vocab = 60_000
    per = 4 if dtype == torch.float32 else 8
    at = torch.arange(vocab)
    x = torch.zeros(4, vocab)
    x[0][(at // per) % 64 == 5] = 9.0
    x[0][per * 5 + 1] = 10.0
    x[1][(at // per) % 256 == 9] = 4.0
    x[1] += at * 2.0 ** -14
    x[2] = at * 2.0 ** -8
    x[3] = torch.sin(at * 0.37) * 5
    x = x.to(dtype)
    for top in (2, 7, 16):
        r = pkg.token_logprobs(x.to(dev), torch.zeros(4, dtype=torch.int64, device=dev), top=top)
        order = x.double().argsort(dim=1, descending=True, stable=True)[:, :top]
        assert torch.equal(r.top_tokens.cpu(), order), top


@types
def test_token_logprobs_masked_and_unsound_rows(pkg, dev, dtype):
    vocab, low, high = 3000, torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn(9, vocab, generator=gen("masked")).to(dtype)
    x[0] = -math.inf                       # nothing left
    x[1] = low                             # masked with the lowest value, all of it
    x[2, 10:] = low                        # and a part of it
    x[3, 5] = math.nan
    x[4, 7] = math.inf
    x[5] = high                            # the largest value everywhere
    x[6] = -math.inf
    x[6, 17] = low                         # one logit, of the lowest value
    x[7, :-1] = -math.inf                  # one logit left
    x[8, 3] = high
    target = torch.full((9,), 5)
    target[6], target[7], target[8] = 17, vocab - 1, 3
    r = pkg.token_logprobs(x.to(dev), target.to(dev), entropy=True, top=3)
    z, lse, lp, ent, _ = logp_want(x, target, 1.0)
    ln = math.log(vocab)
    big = 4 * E * float(high)
    assert r.lse[0] == -math.inf and r.logprobs[0] == -math.inf and r.entropy[0] == 0
    assert bool((r.top_logprobs[0] == -math.inf).all())
    # x - max is exact there, so the log probabilities are a uniform row's
    uniform = (vocab / 256 + 40) * 4 * E * 12
    for row in (1, 5):
        assert abs(float(r.lse[row]) - float(lse[row])) <= big + 12 * E
        assert abs(float(r.logprobs[row]) + ln) <= uniform and abs(float(r.entropy[row]) - ln) <= uniform
        assert r.top_tokens[row].tolist() == [0, 1, 2]
    part = x[2:3].clone()
    part[part == low] = -math.inf
    b = logp_bounds(part, 1.0, lp[2:3])
    check(r.lse[2:3], lse[2:3], b[0], "lse")
    check(r.logprobs[2:3], lp[2:3], b[1], "lp")
    check(r.entropy[2:3], ent[2:3], b[2], "entropy")
    for row in (3, 4):
        assert math.isnan(r.lse[row]) and math.isnan(r.logprobs[row]) and math.isnan(r.entropy[row])
        assert bool(r.top_logprobs[row].isnan().all())
    assert r.top_tokens[4, 0] == 7 and 5 not in r.top_tokens[3].tolist()
    for row in (6, 7, 8):
        assert abs(float(r.logprobs[row])) <= uniform and abs(float(r.entropy[row])) <= uniform
        assert r.top_tokens[row, 0] == target[row]
        assert abs(float(r.lse[row]) - float(lse[row])) <= 4 * E * abs(float(lse[row])) + uniform
    # only NaN, and NaN beside masks: every index once
    y = torch.full((2, 40), math.nan, dtype=dtype)
    y[1, 3:] = -math.inf
    t = pkg.token_logprobs(y.to(dev), torch.zeros(2, dtype=torch.int64, device=dev), top=16).top_tokens
    assert t[0].tolist() == list(range(16)) and t[1].tolist() == list(range(3, 19))


def grad_want(x, target, scale, lse, ent, g, h):
    """The gradient's formula in 64 bits, and the bound of its fp32 evaluation."""
    z = x.double() * scale
    d = z - lse.double()[:, None]
    p = d.exp()
    ok = (target >= 0) & (target < x.shape[1])
    g = torch.where(ok, g.double(), 0.0)[:, None]
    inner = torch.where(p > 0, d + ent.double()[:, None], 0.0)
    h = h.double()[:, None]
    want = -p * (g + h * inner)
    # an exponent's absolute error, e (|z| + |lse|), enters p relatively and log p absolutely (the 1)
    size = p * (g.abs() + h.abs() * (1 + d.abs().nan_to_num(posinf=0) + ent.double().abs()[:, None]))
    hot = torch.zeros_like(z).scatter_(1, torch.where(ok, target, 0)[:, None], g)
    R = torch.where(z.isfinite(), z, 0.0).abs().amax(1, keepdim=True) + lse.double().abs()[:, None].nan_to_num(posinf=0, neginf=0)
    more = size * E * (8 * R + 32) + (hot.abs() + want.abs()) * 4 * E + 2.0 ** -120
    return (want + hot) * scale, more * scale


@types
@pytest.mark.parametrize("rows,vocab", [(1, 1), (4, 3), (3, 8), (5, 65), (4, 2048), (3, 8191), (2, 50304)])
def test_token_logprobs_grad(pkg, dev, dtype, rows, vocab):
    g = gen("lgrad", rows, vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    x[torch.rand(rows, vocab, generator=g) < 0.1] = -math.inf
    x[:, 0] = 0.5
    target = torch.randint(0, vocab, (rows,), generator=g)
    target[-1] = vocab if rows > 1 else 0
    dlp, dent = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    r = pkg.token_logprobs(x.to(dev), target.to(dev), scale=1.3, entropy=True)
    for with_entropy in (True, False):
        h = dent if with_entropy else torch.zeros(rows)
        want, more = grad_want(x, target, 1.3, r.lse.cpu(), r.entropy.cpu(), dlp, h)
        kw = dict(entropy=r.entropy, dentropy=dent.to(dev)) if with_entropy else {}
        got = pkg.token_logprobs_grad(x.to(dev), target.to(dev), r.lse, dlp.to(dev), scale=1.3, **kw)
        assert got.dtype == dtype
        check(got, want, rounded(want, dtype, more), f"lgrad {with_entropy}")
        inplace = x.to(dev)
        assert pkg.token_logprobs_grad(inplace, target.to(dev), r.lse, dlp.to(dev), scale=1.3, out=inplace,
                                       **kw) is inplace
        assert torch.equal(inplace, got)


@types
def test_token_logprobs_strided_rows(pkg, dev, dtype):
    g = gen("strided")
    wide = torch.randn(6, 700, generator=g).to(dtype).to(dev)
    target = torch.randint(0, 333, (6,), generator=g).to(dev)
    for lo in (0, 1, 3, 8):
        view, dense = wide[:, lo:lo + 333], wide[:, lo:lo + 333].contiguous()
        a = pkg.token_logprobs(view, target, entropy=True, top=5)
        b = pkg.token_logprobs(dense, target, entropy=True, top=5)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        g1 = pkg.token_logprobs_grad(dense, target, a.lse, a.lse)
        into = torch.full((6, 700), 5.0, dtype=dtype, device=dev)
        pkg.token_logprobs_grad(view, target, a.lse, a.lse, out=into[:, 350 - lo:683 - lo])
        assert torch.equal(into[:, 350 - lo:683 - lo], g1)
        assert bool((into[:, :350 - lo] == 5).all()) and bool((into[:, 683 - lo:] == 5).all())
    # leading shapes, and no rows
    y = wide[:, :64].contiguous().view(2, 3, 64)
    r = pkg.token_logprobs(y, target.view(2, 3) % 64, top=2)
    assert r.logprobs.shape == (2, 3) and r.top_tokens.shape == (2, 3, 2)
    none = pkg.token_logprobs(y[:0], target.view(2, 3)[:0], entropy=True, top=2)
    assert none.logprobs.shape == (0, 3) and none.top_logprobs.shape == (0, 3, 2)


def test_token_logprobs_of_one_row_and_of_no_vocabulary(pkg, dev):
    x = torch.randn(40, generator=gen("one row")).to(dev)
    target = torch.tensor(7, device=dev)
    r = pkg.token_logprobs(x, target, entropy=True, top=4)
    rows = pkg.token_logprobs(x[None], target[None], entropy=True, top=4)
    assert r.logprobs.shape == () and r.top_tokens.shape == (4,)
    assert all(torch.equal(a, b[0]) for a, b in zip(r, rows))
    d = pkg.token_logprobs_grad(x, target, r.lse, r.entropy)
    assert d.shape == (40,) and torch.equal(d, pkg.token_logprobs_grad(x[None], target[None], rows.lse, rows.entropy)[0])
    none = torch.zeros(3, 0, device=dev)
    t = torch.tensor([0, -100, 5], device=dev)
    r = pkg.token_logprobs(none, t, entropy=True)
    assert r.logprobs.tolist() == [0, 0, 0] and r.entropy.tolist() == [0, 0, 0]
    assert r.lse.tolist() == [-math.inf] * 3
    assert pkg.token_logprobs_grad(none, t, r.lse, r.lse).shape == (3, 0)
    # one token, and rows that are one element apart from being broadcast
    table = torch.randn(5, 12, device=dev)
    assert torch.equal(pkg.embed(torch.tensor(3, device=dev), table), table[3])
    g = pkg.embed_grad(torch.tensor(3, device=dev), table[0], 5)
    assert torch.equal(g[3], table[0]) and int(g.count_nonzero(dim=1).ne(0).sum()) == 1


@types
def test_token_logprobs_grad_of_masked_rows(pkg, dev, dtype):
    vocab, low = 1000, torch.finfo(dtype).min
    x = torch.randn(4, vocab, generator=gen("gmask")).to(dtype)
    x[0] = -math.inf
    x[1] = torch.finfo(torch.bfloat16).min if dtype != torch.float16 else -math.inf
    x[2, 100:] = low
    x[3, 100:] = -math.inf
    target = torch.tensor([5, 5, 5, -100]).to(dev)
    r = pkg.token_logprobs(x.to(dev), target, entropy=True)
    ones = torch.ones(4, device=dev)
    got = pkg.token_logprobs_grad(x.to(dev), target, r.lse, ones, entropy=r.entropy, dentropy=ones).cpu()
    assert not bool(got[:2].any()) and not bool(got[2:, 100:].any()) and bool(got.isfinite().all())
    # an ignored position with a gradient of its own: only the entropy's part
    alone = pkg.token_logprobs_grad(x.to(dev), target, r.lse, ones * 0, entropy=r.entropy, dentropy=ones).cpu()
    assert torch.equal(got[3], alone[3])


def test_token_logprobs_differences(pkg, dev):
    """Central differences of the forward pass against autograd's gradient.  With step t the quotient is off by
    t^2 / 6 of the third derivative (at most 1 for log p, and 20 for the entropy at 30 logits), plus the bounds of both ends over 2 t."""
    g = gen("diff")
    rows, vocab, step = 3, 30, 2.0 ** -6
    x = torch.randn(rows, vocab, generator=g)
    target = torch.tensor([3, 29, -100])
    dlp, dent = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    leaf = x.to(dev).requires_grad_()
    r = pkg.token_logprobs(leaf, target.to(dev), scale=0.7, entropy=True, top=2)
    ((r.logprobs * dlp.to(dev)).sum() + (r.entropy * dent.to(dev)).sum()).backward()
    assert not r.lse.requires_grad and not r.top_logprobs.requires_grad
    lp = logp_want(x, target, 0.7)[2]
    _, b_lp, b_ent = logp_bounds(x, 0.7, lp)
    for j in range(0, vocab, 3):
        ends = []
        for sign in (1, -1):
            y = x.clone()
            y[:, j] += sign * step
            f = pkg.token_logprobs(y.to(dev), target.to(dev), scale=0.7, entropy=True)
            ends.append(f.logprobs.double().cpu() * dlp + f.entropy.double().cpu() * dent)
        quotient = (ends[0] - ends[1]) / (2 * step)
        bound = step ** 2 / 6 * (dlp.abs() + 20 * dent.abs()) + \
            2 * (b_lp * dlp.abs() + b_ent * dent.abs()) / (2 * step) * 2
        check(leaf.grad[:, j], quotient, bound, f"column {j}")
    # only one of the two outputs in the loss
    for pick in ("logprobs", "entropy"):
        one = x.to(dev).requires_grad_()
        f = pkg.token_logprobs(one, target.to(dev), entropy=True)
        getattr(f, pick).sum().backward()
        k = torch.ones(rows, device=dev)
        want = pkg.token_logprobs_grad(one.detach(), target.to(dev), f.lse, k if pick == "logprobs" else k * 0,
                                       **({} if pick == "logprobs" else dict(entropy=f.entropy, dentropy=k)))
        assert torch.equal(one.grad, want)


# ---------------------------------------------------------- gradient lists --

def make_list(g, dev, sizes, kinds):
    """Tensors back to back in one buffer per type, so that they start at any element."""
    out = []
    for i, n in enumerate(sizes):
        t = (torch.randn(n + 3, generator=g) * 10.0 ** (i % 5 - 2)).to(kinds[i % len(kinds)]).to(dev)
        out.append(t[i % 4:i % 4 + n])
    return out


LISTS = [[1], [0], [], [3, 0, 5], [16384], [16385, 7, 16383], [100_000, 1, 2, 3, 65_537], [33] * 1500]


@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s, default=0)}")
@pytest.mark.parametrize("kinds", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=["fp32", "bf16", "fp16", "mix"])
def test_norm_and_clip(pkg, dev, sizes, kinds):
    g = gen("norm", len(sizes), len(kinds))
    grads = make_list(g, dev, sizes, kinds)
    flat = torch.cat([t.double().cpu() for t in grads] + [torch.zeros(1, dtype=torch.float64)])
    norm = float((flat * 0.5).norm())
    got = pkg.grad_norm(grads, grad_scale=0.5)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - norm) <= 2 * E * norm
    most = float((flat * 0.5).abs().max())
    assert float(pkg.grad_norm(grads, math.inf, grad_scale=-0.5)) == most
    for limit in (norm / 3 + 1e-3, norm * 2 + 1):
        by = 0.5 * min(1.0, limit / (norm + 1e-6))
        for out in TYPES:
            outs = make_list(g, dev, sizes, [out])
            got = pkg.clip_grads(grads, limit, grad_scale=0.5, out=outs)
            assert abs(float(got) - norm) <= 2 * E * norm
            for t, o in zip(grads, outs):
                want = t.double().cpu() * by
                check(o, want, rounded(want, out, want.abs() * 8 * E), f"clip to {out}")
        same = [t.clone() for t in grads]
        pkg.clip_grads(same, limit, grad_scale=0.5)
        for t, o in zip(grads, same):
            want = t.double().cpu() * by
            check(o, want, rounded(want, t.dtype, want.abs() * 8 * E), "clip in place")


@types
def test_norm_and_clip_of_many_pieces(pkg, dev, dtype):
    """More pieces than the launches of a short list take: 34 M elements, the last tensors odd."""
    sizes = [33_600_001, 17, 400_003]
    buf = torch.randn(sum(sizes) + 1, generator=gen("many"), dtype=torch.float32).to(dtype).to(dev)[1:]
    grads = list(buf.split(sizes))
    norm = float((buf.double() * 0.25).norm())
    lst = pkg.GradList(grads)
    assert abs(float(lst.norm(grad_scale=0.25)) - norm) <= 2 * E * norm
    assert float(lst.norm(math.inf, grad_scale=0.25)) == float((buf.double() * 0.25).abs().max())
    by = 0.25 * 3.0 / (norm + 1e-6)
    for out in TYPES:
        into = torch.full((sum(sizes) + 6,), 5.0, dtype=out, device=dev)
        got = pkg.GradList(grads, list(into[3:-3].split(sizes))).clip(3.0, grad_scale=0.25)
        assert abs(float(got) - norm) <= 2 * E * norm
        want = buf.double() * by
        off = (into[3:-3].double() - want).abs() - (want.abs() * (UNIT[out] + 8 * E) * 1.01 + TINY[out])
        assert float(off.max()) <= 0, out
        assert bool((into[:3] == 5).all()) and bool((into[-3:] == 5).all())
    kept = buf.clone()
    lst.clip(1e6)
    assert torch.equal(buf, kept)
    given = torch.tensor(100.0, device=dev)
    assert float(lst.clip(1.0, norm=given)) == 100.0
    want = kept.double() * 0.01
    assert float(((buf.double() - want).abs() - (want.abs() * (UNIT[dtype] + 8 * E) * 1.01 + TINY[dtype])).max()) <= 0
    buf[-1] = math.inf
    kept = buf.clone()
    assert float(lst.clip(1.0)) == math.inf and torch.equal(buf, kept)


def test_norm_at_the_ends_of_the_range(pkg, dev):
    big = torch.full((1000,), 1e30, device=dev)             # the squares are past fp32
    assert abs(float(pkg.grad_norm([big])) / (1e30 * math.sqrt(1000)) - 1) <= 4 * E
    small = torch.full((1000,), 1e-30, device=dev)
    assert abs(float(pkg.grad_norm([small])) / (float(small[0]) * math.sqrt(1000)) - 1) <= 4 * E
    assert float(pkg.grad_norm([torch.full((4,), 3e38, device=dev)])) == math.inf
    for bad in (math.nan, math.inf, -math.inf):
        for kind in TYPES:
            g = [torch.ones(5000, dtype=kind, device=dev), torch.ones(20_000, dtype=kind, device=dev)]
            g[1][17_777] = bad
            for norm_type in (2, math.inf):
                n = float(pkg.grad_norm(g, norm_type))
                assert math.isnan(n) if math.isnan(bad) else n == math.inf
            kept = [t.clone() for t in g]
            n = pkg.clip_grads(g, 1.0)
            assert not math.isfinite(n)
            assert all(torch.equal(a.nan_to_num(nan=5.0), b.nan_to_num(nan=5.0)) for a, b in zip(g, kept))
            outs = [torch.empty_like(t) for t in g]
            pkg.clip_grads(g, 1.0, grad_scale=0.5, out=outs)
            assert all(torch.equal((a * 0.5).nan_to_num(nan=5.0), b.nan_to_num(nan=5.0)) for a, b in zip(g, outs))


def test_clip_leaves_a_small_norm_alone_and_takes_a_given_one(pkg, dev):
    g = [torch.randn(777, generator=gen("keep")).to(dev), torch.zeros(5, dtype=torch.bfloat16, device=dev)]
    kept = [t.clone() for t in g]
    lst = pkg.GradList(g)
    n = lst.clip(1e9)
    assert all(torch.equal(a, b) for a, b in zip(g, kept)) and float(n) == float(lst.norm())
    given = torch.tensor(50.0, device=dev)
    assert float(lst.clip(5.0, norm=given)) == 50.0
    by = torch.tensor(5.0) / (torch.tensor(50.0) + 1e-6)
    want = kept[0].double().cpu() * float(by)
    check(g[0], want, rounded(want, torch.float32, want.abs() * 4 * E), "given")
    # two ranks' norms, joined
    a, b = pkg.grad_norm(kept[:1]), pkg.grad_norm([kept[0] * 2])
    joined = torch.stack([a, b]).square().sum().sqrt()
    pkg.clip_grads(kept, 0.5, norm=joined)
    assert abs(float(pkg.grad_norm(kept)) - 0.5 * float(a) / float(joined)) <= 1e-5


def test_grad_list_refusals(pkg, dev):
    ok = torch.zeros(8, device=dev)
    for grads, out in (([ok.view(2, 4).t()], None), ([ok.double()], None), ([ok], [ok[:4]]), ([ok], []),
                       ([ok], [ok.double()])):
        with pytest.raises(ValueError):
            pkg.GradList(grads, out)
    lst = pkg.GradList([ok])
    for call in (lambda: lst.norm(1), lambda: lst.norm(grad_scale=math.inf), lambda: lst.clip(0.0),
                 lambda: lst.clip(1.0, norm=torch.ones(2, device=dev)), lambda: lst.clip(1.0, norm=torch.ones(1)),
                 lambda: lst.clip(1.0, norm=ok.double()[:1])):
        with pytest.raises(ValueError):
            call()


def test_memory_that_is_written_and_read(pkg, dev):
    """Results over their own operands are refused where a value could be read after it was written;
    the gradient over its logits, and columns beside each other, are not."""
    buf = torch.randn(40, 64, device=dev)
    tok = torch.arange(20, device=dev)
    for call in (lambda: pkg.embed(tok, buf[:20], out=buf[:20]),
                 lambda: pkg.embed(tok, buf[:20, :32], out=buf.view(-1)[16:656].view(20, 32)),
                 lambda: pkg.embed_grad(tok, buf[:20], 20, out=buf[10:30]),
                 lambda: pkg.embed_grad(tok, buf[:20, :32], 20, out=buf[:20, 16:48]),
                 lambda: pkg.token_logprobs_grad(buf[:20], tok, buf[0, :20], buf[0, :20], out=buf[1:21]),
                 lambda: pkg.GradList([buf[:20], buf[10:30]]), lambda: pkg.GradList([buf, buf]),
                 lambda: pkg.GradList([buf[:20]], out=[buf[1:21]]),
                 lambda: pkg.GradList([buf[:20], buf[20:]], out=[buf[20:], buf[:20]]),
                 lambda: pkg.GradList([buf[:10].bfloat16(), buf[20:]], out=[buf[25:35], buf.new_zeros(20, 64)])):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    # neighbours, the same place, and reads that overlap
    left, right = buf[:20, :32], buf[:20, 32:]
    want = pkg.embed_grad(tok, left, 20)
    assert torch.equal(pkg.embed_grad(tok, left, 20, out=right), want)
    outs = [torch.empty(20, 64, device=dev) for _ in range(2)]
    assert float(pkg.GradList([buf[:20], buf[10:30]], out=outs).clip(1e9)) > 0
    assert torch.equal(outs[1], buf[10:30])
    pkg.GradList([buf[:20], buf[20:]], out=[buf[:20], buf[20:]]).clip(1e9)
    pkg.GradList([buf[:20], buf[20:], buf[:0]]).clip(1e9)


def test_a_second_derivative_is_refused(pkg, dev):
    table = torch.randn(5, 8, device=dev, requires_grad=True)
    x = torch.randn(3, 20, device=dev, requires_grad=True)
    tok = torch.tensor([0, 1, 2], device=dev)
    for out, leaf in ((pkg.embed(tok, table), table), (pkg.token_logprobs(x, tok).logprobs, x)):
        (g,) = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


def test_refusals_on_device(pkg, dev):
    table, tok = torch.zeros(10, 8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    x, lse = torch.zeros(3, 50, device=dev), torch.zeros(3, device=dev)
    dout = torch.zeros(3, 8, device=dev)
    for call in (lambda: pkg.embed(tok.float(), table), lambda: pkg.embed(tok, table.t()),
                 lambda: pkg.embed(tok, table[0]), lambda: pkg.embed(tok, table, out=dout[:2]),
                 lambda: pkg.embed(tok, table, out=dout.bfloat16()), lambda: pkg.embed(tok.cpu(), table),
                 lambda: pkg.embed(tok.expand(2, 3), table),
                 lambda: pkg.embed_grad(tok, dout[:2], 10), lambda: pkg.embed_grad(tok, dout, -1),
                 lambda: pkg.embed_grad(tok, dout, 10, accumulate=True),
                 lambda: pkg.embed_grad(tok, dout, 10, dtype=torch.bfloat16),
                 lambda: pkg.embed_grad(tok, dout[:1].expand(3, 8), 10),
                 lambda: pkg.token_logprobs(x, tok.int()), lambda: pkg.token_logprobs(x, tok[:2]),
                 lambda: pkg.token_logprobs(x.t(), tok), lambda: pkg.token_logprobs(x, tok, top=17),
                 lambda: pkg.token_logprobs(x[:, :4], tok, top=5), lambda: pkg.token_logprobs(x, tok, top=-1),
                 lambda: pkg.token_logprobs_grad(x, tok, lse, lse.double()),
                 lambda: pkg.token_logprobs_grad(x, tok, lse[:2], lse),
                 lambda: pkg.token_logprobs_grad(x, tok, lse, lse, entropy=lse),
                 lambda: pkg.token_logprobs_grad(x, tok, lse, lse, out=x[:, :49])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError, match="gradients"):
        pkg.embed(tok, table.clone().requires_grad_(), out=dout)


# ------------------------------------------------------- streams and graphs --

def test_on_a_caller_stream(pkg, dev):
    """Each operator on a stream of its own behind a long kernel, the inputs made there, the results read
    after it; memory of dropped results is not handed out before that stream is done."""
    side = torch.cuda.Stream(dev)
    g = gen("streams")
    table = torch.randn(500, 256, generator=g).to(dev)
    tok = torch.randint(0, 500, (4000,), generator=g).to(dev)
    x = torch.randn(64, 5000, generator=g).to(dev)
    target = torch.randint(0, 5000, (64,), generator=g).to(dev)
    want = [pkg.embed(tok, table), pkg.embed_grad(tok, table[tok], 500), *pkg.token_logprobs(x, target, entropy=True, top=4),
            pkg.grad_norm([table, x])]
    r = pkg.token_logprobs(x, target)
    want.append(pkg.token_logprobs_grad(x, target, r.lse, r.lse))
    lst = pkg.GradList([table, x])
    rows = table[tok]
    torch.cuda.synchronize()
    a = torch.randn(4096, 4096, device=dev)
    for _ in range(3):
        with torch.cuda.stream(side):
            for _ in range(4):
                a = a @ a * 1e-2
        got = [pkg.embed(tok, table, stream=side), pkg.embed_grad(tok, rows, 500, stream=side),
               *pkg.token_logprobs(x, target, entropy=True, top=4, stream=side), lst.norm(stream=side)]
        got.append(pkg.token_logprobs_grad(x, target, r.lse, r.lse, stream=side))
        junk = [torch.full((4000, 256), 3.0, device=dev) for _ in range(4)]
        # the result's block goes back while the current stream has yet to read it
        torch.cuda.current_stream().wait_stream(side)
        kept = got[0] + 0
        got[0] = kept
        again = pkg.embed(tok, table, scale=2.0, stream=side)
        side.synchronize()
        torch.cuda.current_stream().synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        del junk, got, kept, again
    with torch.cuda.stream(side):   # torch's current stream is another than the list was made on
        n = lst.norm()
    side.synchronize()
    assert float(n) == float(want[-2])


def test_captured_in_a_graph(pkg, dev):
    """A step's operators recorded once and replayed over new inputs, eager work between the replays."""
    g = gen("graph")
    table = torch.randn(300, 64, generator=g).to(dev)
    tok = torch.randint(0, 300, (5000,), generator=g).to(dev)
    x = torch.randn(32, 4000, generator=g).to(dev)
    target = torch.randint(0, 4000, (32,), generator=g).to(dev)
    lst = pkg.GradList([table, x])

    def step():
        e = pkg.embed(tok, table)
        d = pkg.embed_grad(tok, e, 300)
        r = pkg.token_logprobs(x, target, entropy=True, top=3)
        gx = pkg.token_logprobs_grad(x, target, r.lse, r.logprobs, entropy=r.entropy, dentropy=r.lse)
        return [e, d, *r, gx, lst.norm()]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        tok.copy_(torch.randint(0, 300, (5000,), generator=g))
        x.copy_(torch.randn(32, 4000, generator=g))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want)), k


def test_offsets_past_32_bits(pkg, dev):
    """Logits and tables of more than 2^32 elements: the last rows are where they belong."""
    rows, vocab = 70_000, 65_536
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=dev)
    x[-1, 5] = 9.0
    x[-1, vocab - 1] = 8.0
    target = torch.full((rows,), 5, device=dev)
    r = pkg.token_logprobs(x, target, top=2)
    assert r.top_tokens[-1].tolist() == [5, vocab - 1] and r.top_tokens[-2].tolist() == [0, 1]
    d = pkg.token_logprobs_grad(x, target, r.lse, torch.ones(rows, device=dev), out=x)
    p = math.exp(float(r.logprobs[-1]))
    assert abs(float(d[-1, 5]) - (1 - p)) <= 2.0 ** -8 * (1 - p) and abs(float(d[0, 6]) + 1 / vocab) <= 2.0 ** -8 / vocab
    x.zero_()
    x[-1] = 2.0
    got = pkg.embed(torch.tensor([rows - 1, 0, rows], device=dev), x, scale=3.0)
    assert bool((got[0] == 6).all()) and not bool(got[1:].any())
    tok = torch.arange(rows, device=dev).flip(0)
    grad = pkg.embed_grad(tok, x, 3, vocab_start=0, dtype=torch.bfloat16)
    assert bool((grad[0] == 2).all()) and not bool(grad[1:].any())


def test_example_trains_saves_and_loads():
    """The example's loop: the loss falls, and the state rebuilt from the slices answers with the same
    bits (the example raises otherwise)."""
    path = os.path.join(ROOT, "megatron-lm_amd", "examples", "train_step.py")
    spec = importlib.util.spec_from_file_location("train_step_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(60) < 3.0   # ln 512 = 6.2 at the start
