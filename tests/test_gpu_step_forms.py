"""The forms that the step operators' kernels take by their rules on sizes, on both sides of each: lanes per row of
logits, streamed rows of logits, the search for the likeliest tokens, streamed rows of an embedding."""
import math

import pytest
import torch

from test_gpu_step import E, gen, grad_want, logp_want, rounded, types

pytestmark = pytest.mark.gpu


def check(got, want, bound, what):
    """test_gpu_step.check on the device."""
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    sane = want.isfinite()
    assert bool((sane | want.isnan() | (got == want)).all()), f"{what}: infinities"
    off = torch.where(sane, (got - want).abs() - bound, -1.0)
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} over, by {float(off.max()):.3g}"


def logits(dev, rows, vocab, dtype, key, pad=0):
    """Normal logits with a tenth masked, made on the device (the shapes are large), rows `pad` elements apart."""
    g = torch.Generator(device=dev)
    g.manual_seed(rows * 1009 + vocab + key)
    x = torch.empty(rows, vocab + pad, device=dev).normal_(0.0, 3.0, generator=g)
    x[torch.rand(rows, vocab + pad, generator=g, device=dev) < 0.1] = -math.inf
    x[:, 0] = 1.0
    target = torch.randint(-1, vocab + 1, (rows,), generator=g, device=dev)
    return x.to(dtype)[:, :vocab], target


def bounds(x, scale, lp):
    """test_gpu_step.logp_bounds for a row of as few as 128 lanes."""
    R = torch.where(x.isfinite(), x.double() * scale, 0.0).abs().amax(1)
    s = (x.shape[1] / 128 + 28 + 4 + 4 * (R + 1)) * E
    return s + 4 * E * (R + 12), s + 4 * E * (lp.abs() + 12), (s * 4 + 16 * E) * (R + 12)


def forward(pkg, x, target, scale, tops, entropies=(False, True)):
    z, lse, lp, ent, _ = logp_want(x, target, scale)
    b_lse, b_lp, b_ent = bounds(x, scale, lp)
    order = x.double().argsort(dim=1, descending=True, stable=True)[:, :max(tops)] if max(tops) else None
    for entropy in entropies:
        for top in tops:
            r = pkg.token_logprobs(x, target, scale=scale, entropy=entropy, top=top)
            check(r.lse, lse, b_lse, "lse")
            check(r.logprobs, lp, b_lp, "logprobs")
            if entropy:
                check(r.entropy, ent, b_ent, "entropy")
            if top:
                assert torch.equal(r.top_tokens, order[:, :top])
                want = z.gather(1, order[:, :top]) - lse[:, None]
                check(r.top_logprobs, want, b_lp[:, None] + 4 * E * want.abs().nan_to_num(posinf=0), "top")
    return r


@pytest.mark.parametrize("rows", [1024, 1025])
@pytest.mark.parametrize("dtype,vocab", [(t, v) for t in (torch.bfloat16, torch.float16) for v in (1, 7, 1003, 16376, 16384)] +
                         [(torch.float32, v) for v in (1, 7, 1003, 8184, 8192)])
def test_lanes_per_row(pkg, dev, dtype, vocab, rows):
    """1024 rows and fewer, and rows of 2048 groups of 16 bytes and more, take 512 lanes; others 128."""
    x, target = logits(dev, rows, vocab, dtype, 1)
    forward(pkg, x, target, 0.8, sorted({0, 1, min(16, vocab)}))


@types
def test_the_search_of_short_rows(pkg, dev, dtype):
    """More candidates than there is room for, in rows of 128 lanes: three of every 64 groups hold all large logits, equal
    ones or not."""
    vocab = 16_000 if dtype != torch.float32 else 8000
    at = torch.arange(vocab, device=dev)
    group = at // (16 // dtype.itemsize)
    x, target = logits(dev, 1030, vocab, dtype, 2)
    x[::2] = torch.where((group % 64 >= 5) & (group % 64 < 8), 9.0, torch.zeros(vocab, device=dev)).to(dtype)
    x[1::4] = torch.where((group % 128 == 70) | (group % 128 == 100) | (group % 64 == 9), 8.0 + (at % 97) / 64, x[1::4].float()).to(dtype)
    forward(pkg, x, target, 1.0, (2, 16), (True,))


@pytest.mark.parametrize("dtype,rows,vocab,pad", [
    (torch.bfloat16, 1100, 65_537, 0), (torch.float16, 1030, 65_536, 7), (torch.float32, 530, 65_537, 3),
    (torch.bfloat16, 20_011, 4001, 0), (torch.float16, 17_000, 4008, 8), (torch.float32, 17_000, 2003, 0)],
    ids=["bf16", "fp16", "fp32", "bf16 short", "fp16 short", "fp32 short"])
def test_streamed_logits(pkg, dev, dtype, rows, vocab, pad):
    """Logits of more than 128 MiB, long rows and short ones, dense and strided: forward, alternatives and the gradient
    with and without the entropy's."""
    x, target = logits(dev, rows, vocab, dtype, 3, pad)
    assert x.numel() * dtype.itemsize > 128 << 20
    r = forward(pkg, x, target, 0.8, (0, 5))
    g = torch.Generator(device=dev)
    g.manual_seed(rows)
    dlp, dent = (torch.randn(rows, generator=g, device=dev) for _ in range(2))
    for with_entropy in (True, False):
        h = dent if with_entropy else dent * 0
        want, more = grad_want(x, target, 0.8, r.lse, r.entropy, dlp, h)
        kw = dict(entropy=r.entropy, dentropy=dent) if with_entropy else {}
        got = pkg.token_logprobs_grad(x, target, r.lse, dlp, scale=0.8, **kw)
        check(got, want, rounded(want, dtype, more), f"gradient {with_entropy}")
    torch.cuda.empty_cache()


@types
@pytest.mark.parametrize("hidden", [1033, 2048])
def test_streamed_embed(pkg, dev, dtype, hidden):
    """Results on both sides of 64 MiB, in rows of at least a KiB."""
    table = torch.randn(501, hidden, generator=gen("wide", hidden)).to(dtype).to(dev)
    edge = (64 << 20) // (hidden * dtype.itemsize)
    for n in (edge - 1, edge, edge + 1, edge + 777):
        tok = (torch.arange(n, device=dev) * 31) % 530
        got = pkg.embed(tok, table, scale=0.5)
        want = torch.where(tok[:, None] < 501, table[tok.clamp(max=500)] * 0.5, 0.0)
        assert torch.equal(got, want)
