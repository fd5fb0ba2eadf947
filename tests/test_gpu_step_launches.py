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
