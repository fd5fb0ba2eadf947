"""embed_grad of more than 2^20 tokens, whose sort takes several tiles a workgroup."""
import pytest
import torch

from test_gpu_step import E, TINY, UNIT, gen

pytestmark = pytest.mark.gpu

TILE, SPANS = 2048, 512


@pytest.mark.parametrize("n", [TILE * SPANS, TILE * SPANS + 1, TILE * (SPANS * 2 - 1) + 5, TILE * SPANS * 2 + 1, 3_456_789])
@pytest.mark.parametrize("vocab,hidden", [(300, 3), (50_304, 2), (262_145, 1)])
def test_embed_grad_of_many_tokens(pkg, dev, n, vocab, hidden):
    """Both sides of the sizes where a workgroup gets another tile; vocabularies of two digits and three, one past the
    bits of the rows that occur; one token on every seventh position, some outside."""
    g = gen("many", n, vocab)
    tok = (torch.rand(n, generator=g) ** 3 * (vocab + 2)).long() - 1
    tok[::7] = vocab // 2
    dout = torch.randn(n, hidden, generator=g).bfloat16()
    # (on the host: the device's index_add_ would wait for each of the many additions to one place)
    here = (tok >= 0) & (tok < vocab)
    rows, some = tok[here], dout[here].double()
    want = torch.zeros(vocab, hidden, dtype=torch.float64).index_add_(0, rows, some)
    size = torch.zeros_like(want).index_add_(0, rows, some.abs())
    count = torch.zeros(vocab, 1, dtype=torch.float64).index_add_(0, rows, torch.ones_like(some[:, :1]))
    want, size, count, tok, dout = (t.to(dev) for t in (want, size, count, tok, dout))
    got = pkg.embed_grad(tok, dout, vocab)
    # a run is summed by tiles of 32 tokens, their sums 8 at a time by 8 waves: the additions behind one another
    adds = 32 + count.div(32).ceil() + 2 + 8
    bound = want.abs() * UNIT[torch.float32] * 1.01 + TINY[torch.float32] + adds.minimum(count + 2) * E * size * 1.01
    assert bool(((got.double() - want).abs() <= bound).all())
    assert not bool(got[count[:, 0] == 0].any())
    assert torch.equal(pkg.embed_grad(tok.int(), dout, vocab), got)
    keep = torch.full((vocab, hidden), 2.0, device=dev)
    pkg.embed_grad(tok, dout, vocab, out=keep, accumulate=True)
    assert bool((keep[count[:, 0] == 0] == 2).all())
    assert bool(((keep.double() - 2 - want).abs() <= bound + (want.abs() + 2) * E * 1.01).all())


def test_equal_tokens_stay_in_order(pkg, dev):
    """The positions of a token are added in ascending order: the sums are those of the same tokens' rows at the same
    places of a short list, where the sort is another."""
    few, times = 40, 30_011
    n = few * times
    tok = torch.arange(n, device=dev) % few                  # its positions: v, v + 40, ...
    dout = torch.randn(n, 1, generator=gen("order")).to(dev)
    got = pkg.embed_grad(tok, dout, few)
    grouped = pkg.embed_grad(torch.arange(few, device=dev).repeat_interleave(times), dout.view(times, few).t().reshape(n, 1), few)
    assert torch.equal(got, grouped)
