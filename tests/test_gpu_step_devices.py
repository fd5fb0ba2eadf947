"""Step operators and flat-shard calls on tensors of a device that is not the current one.  One device shows only that the calls keep the
current one; the rest needs two."""
import pytest
import torch

from test_gpu_step import gen

pytestmark = pytest.mark.gpu


def everything(pkg, dev):
    g = gen("devices")
    table = torch.randn(70, 40, generator=g).to(dev)
    tok = torch.randint(0, 80, (9000,), generator=g).to(dev)
    x = torch.randn(30, 500, generator=g).to(dev)
    target = torch.randint(0, 500, (30,), generator=g).to(dev)
    e = pkg.embed(tok, table)
    r = pkg.token_logprobs(x, target, entropy=True, top=3)
    d = pkg.token_logprobs_grad(x, target, r.lse, r.logprobs)
    lst = pkg.GradList([table, x])
    out = [e, pkg.embed_grad(tok, e, 70), *r, d, lst.norm(), lst.clip(0.5), table, x, pkg.grad_norm([x])]
    leaf = table.detach().requires_grad_()
    pkg.token_logprobs(pkg.embed(tok[:30], leaf), target % 40).logprobs.sum().backward()
    shards = [torch.randint(0, 256, (5000,), dtype=torch.uint8, generator=g).to(dev) for _ in range(4)]
    coded = [pkg.xor_encode(shards), *pkg.rs_encode(shards, 2)]
    return [t.cpu() for t in out + coded + [leaf.grad]]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_on_a_device_that_is_not_current(pkg, dev):
    want = everything(pkg, torch.device("cuda", 0))
    with torch.cuda.device(0):
        got = everything(pkg, torch.device("cuda", 1))
        assert torch.cuda.current_device() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_current_device_stays(pkg, dev):
    before = torch.cuda.current_device()
    assert len(everything(pkg, dev)) == 17
    assert torch.cuda.current_device() == before
