"""Step operators past the 2^32 lanes that one launch takes, and their neighbours on both sides of its end."""
import numpy as np
import pytest
import torch

from test_gpu_step import gen

pytestmark = pytest.mark.gpu


def room(gib):
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    if free < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory, {free >> 30} are free")


def test_embed_of_more_tokens_than_a_launch(pkg, dev):
    """2^26 rows of more than 2 KiB: a launch ends at row 2^26 - 4."""
    room(160)
    hidden, n = 1033, (1 << 26) + 5
    table = torch.randn(90, hidden, generator=gen("launches")).bfloat16().to(dev)
    tok = (torch.arange(n, dtype=torch.int32, device=dev) * 7) % 97        # some of them outside
    out = pkg.embed(tok, table)
    rows = torch.cat([torch.arange(0, n, 100_003), torch.arange((1 << 26) - 40, n)]).to(dev)
    ids = tok[rows].long()
    want = torch.where(ids[:, None] < 90, table[ids.clamp(max=89)], 0.0)
    assert torch.equal(out[rows], want)
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("entropy,top", [(False, 0), (True, 2)])
def test_logprobs_of_more_rows_than_a_launch(pkg, dev, entropy, top):
    """More rows of three logits than a launch takes in any form; the gradient's rows run over two and three launches."""
    room(16)
    n, few = (1 << 25) + 7, 1013
    base = torch.randn(few, 3, generator=gen("rows")).to(dev)
    goal = torch.randint(-1, 4, (few,), generator=gen("goals")).to(dev)
    at = torch.arange(n, device=dev) % few
    x, target = base.bfloat16()[at], goal[at]
    want = pkg.token_logprobs(base.bfloat16(), goal, entropy=entropy, top=top)
    r = pkg.token_logprobs(x, target, entropy=entropy, top=top)
    for got, some in zip(r, want):
        if some is not None:
            assert torch.equal(got, some[at])
    kw = dict(entropy=r.entropy, dentropy=r.lse) if entropy else {}
    some = dict(entropy=want.entropy, dentropy=want.lse) if entropy else {}
    d = pkg.token_logprobs_grad(base.bfloat16(), goal, want.lse, want.logprobs, **some)
    assert torch.equal(pkg.token_logprobs_grad(x, target, r.lse, r.logprobs, **kw), d[at])
    torch.cuda.empty_cache()


def test_clip_of_more_pieces_than_a_launch(pkg, dev):
    """2^21 and some small tensors, as the C entry point takes them: in place and into another type, the norm given or not."""
    lib = pkg._lib.lib()
    n = (1 << 21) + 9
    src = torch.randn(n, 3, generator=gen("pieces")).to(dev)
    dst = torch.zeros(n, 3, dtype=torch.bfloat16, device=dev)
    item = np.dtype([("src", "u8"), ("dst", "u8"), ("n", "u4"), ("src_type", "u2"), ("dst_type", "u2")])
    items = np.zeros(n, item)
    items["src"] = src.data_ptr() + 12 * np.arange(n, dtype=np.uint64)
    items["dst"] = dst.data_ptr() + 6 * np.arange(n, dtype=np.uint64)
    items["n"], items["src_type"], items["dst_type"] = 3, 0, 1
    work = torch.empty(8192, dtype=torch.uint8, device=dev)
    norm = torch.zeros((), device=dev)
    given = torch.tensor(50.0, device=dev)
    stream = torch.cuda.current_stream(dev).cuda_stream

    def clip(items, most, given):
        up = torch.from_numpy(items.view(np.uint8)).to(dev)
        norm.zero_()
        assert lib.ec_grad_clip(up.data_ptr(), n, 1.0, 2, most, given, work.data_ptr(), norm.data_ptr(), stream) == 0
        torch.cuda.synchronize()

    total = float(src.double().norm())
    clip(items, total / 4, None)
    assert abs(float(norm) - total) <= 2 ** -22 * total
    want = src.double() / 4
    assert bool(((dst.double() - want).abs() <= want.abs() * 2 ** -8 * 1.01 + 1e-7).all())
    clip(items, 5.0, given.data_ptr())
    assert float(norm) == 50.0
    want = src.double() / 10
    assert bool(((dst.double() - want).abs() <= want.abs() * 2 ** -8 * 1.01 + 1e-7).all())
    items["dst"], items["dst_type"] = items["src"], 0
    kept = src.clone()
    clip(items, total / 2, None)
    assert bool(((src.double() - kept.double() / 2).abs() <= kept.double().abs() * 2 ** -22 + 1e-7).all())
