"""What a step operator writes into a caller's tensor is seen by autograd, as torch's own in-place operations are."""
import pytest
import torch

from test_gpu_step import gen

pytestmark = pytest.mark.gpu

TOK = torch.arange(6)


def saved(dev, *shape):
    """(a tensor, a loss whose backward pass has saved it)"""
    t = torch.randn(*shape, generator=gen("saved", shape)).to(dev)
    weight = torch.ones(*shape, device=dev, requires_grad=True)
    return t, (t * weight).sum()


def calls(pkg, dev):
    rows = torch.randn(6, 8, device=dev)
    x = torch.randn(6, 8, device=dev)
    tok = TOK.to(dev)
    r = pkg.token_logprobs(x, tok)
    return {
        "embed": lambda t: pkg.embed(tok, rows, out=t),
        "embed_grad": lambda t: pkg.embed_grad(tok, rows, 6, out=t),
        "accumulate": lambda t: pkg.embed_grad(tok, rows, 6, out=t, accumulate=True),
        "logits": lambda t: pkg.token_logprobs_grad(x, tok, r.lse, r.lse, out=t),
        "in place": lambda t: pkg.token_logprobs_grad(t, tok, r.lse, r.lse, out=t),
        "clip": lambda t: pkg.GradList([rows, t]).clip(1e-3),
        "clip out": lambda t: pkg.clip_grads([x], 1e-3, out=[t]),
        "part": lambda t: pkg.clip_grads([x[2:4]], 1e-3, out=[t[3:5]]),
    }


@pytest.mark.parametrize("name", ["embed", "embed_grad", "accumulate", "logits", "in place", "clip", "clip out", "part"])
def test_a_saved_tensor_that_is_written_is_noticed(pkg, dev, name):
    call = calls(pkg, dev)[name]
    t, loss = saved(dev, 6, 8)
    call(t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():      # tensors without a version
        call(torch.zeros(6, 8, device=dev))


def test_logits_overwritten_before_their_backward_pass(pkg, dev):
    x = torch.randn(6, 50, device=dev, requires_grad=True)
    logits = x * 1.0
    r = pkg.token_logprobs(logits, TOK.to(dev))
    d = logits.detach()
    pkg.token_logprobs_grad(d, TOK.to(dev), r.lse, torch.ones_like(r.lse), out=d)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()


def test_what_is_only_read_keeps_its_version(pkg, dev):
    t, loss = saved(dev, 6, 8)
    tok = TOK.to(dev)
    r = pkg.token_logprobs(t, tok, entropy=True, top=2)
    pkg.token_logprobs_grad(t, tok, r.lse, r.lse)
    pkg.embed(tok, t)
    pkg.embed_grad(tok, t, 6)
    lst = pkg.GradList([t], out=[torch.empty_like(t)])
    lst.norm()
    lst.clip(1.0)
    pkg.grad_norm([t])
    loss.backward()


def test_views_of_one_buffer(pkg, dev):
    """A list of a buffer's pieces: the buffer, its other views and what shares its version were written; others were not."""
    flat = torch.randn(40, device=dev)
    other = torch.randn(8, device=dev)
    pieces = list(flat.split([8, 20, 12])) + [flat.detach()[:0]]
    lst = pkg.GradList(pieces + [other])
    for t in (flat, flat[30:], flat.view(5, 8), pieces[1], flat.detach(), other):
        weight = torch.ones_like(t, requires_grad=True)
        loss = (t * weight).sum()
        lst.clip(1e-3)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    kept, loss = saved(dev, 8)
    lst.clip(1e-3)
    loss.backward()
    before = flat._version
    lst.norm()
    assert flat._version == before
