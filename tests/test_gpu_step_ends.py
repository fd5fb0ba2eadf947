"""The log probabilities' entropy where logits are large: finite masks.  Bounds as in test_gpu_step.py."""
import math

import numpy as np
import pytest
import torch

from test_gpu_step import E, check, gen, logp_bounds, logp_want

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- entropy --

@pytest.mark.parametrize("scale", [1.0, 1 / 0.6, 1 / 0.2, 1 / 1.2, 1 / 0.55], ids=lambda s: f"{s:.3g}")
@pytest.mark.parametrize("mask", [-1e9, -2e9, -1e10])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_entropy_behind_finite_masks(pkg, dev, dtype, mask, scale):
    """Rows masked with a finite value, whole groups of it before a lane's first live logit: the product of
    mask and scale is rounded by up to 2^7 there, which the running sums of a lane start from."""
    g = gen("finite masks")
    vocab = 30_011
    x = (torch.randn(5, vocab, generator=g) * 2).to(dtype)
    live = torch.ones(5, vocab, dtype=torch.bool)
    live[0, :9000] = False                                   # the first groups of every lane
    live[1] = torch.arange(vocab) % 64 < 8                   # a few lanes' groups
    live[2] = torch.arange(vocab) >= vocab - 3               # only the row's end
    live[3] = torch.arange(vocab) // 4096 % 2 == 1           # masks between
    live[4] = torch.rand(vocab, generator=g) < 0.001
    live[4, 20_000] = True
    x = torch.where(live, x, torch.tensor(mask).to(dtype))
    target = torch.tensor([9000, 64, vocab - 1, 4096, 20_000])
    part = torch.where(live, x, -math.inf)
    _, lse, lp, ent, p = logp_want(part, target, scale)
    b_lse, b_lp, b_ent = logp_bounds(part, scale, lp)
    for top in (0, 3):
        r = pkg.token_logprobs(x.to(dev), target.to(dev), scale=scale, entropy=True, top=top)
        check(r.lse, lse, b_lse, "lse")
        check(r.logprobs, lp, b_lp, "logprobs")
        check(r.entropy, ent, b_ent, "entropy")
    ones = torch.ones(5, device=dev)
    got = pkg.token_logprobs_grad(x.to(dev), target.to(dev), r.lse, ones, scale=scale, entropy=r.entropy, dentropy=ones)
    assert bool(got.isfinite().all()) and not bool(got.cpu()[~live].any())


@pytest.mark.parametrize("vocab", [2, 5, 16])
def test_entropy_of_a_uniform_row_past_the_sums_range(pkg, dev, vocab):
    """A row of one large value whose product with log2 e is rounded by about 2^7: the sum of the exponentials, or
    only the weighted one of the entropy, is past fp32."""
    c = np.float64(np.float32(1.44269504088896340736))
    values = np.float32(-1.5e9) - np.arange(0, 1 << 14, dtype=np.float32) * np.float32(128)
    off = values.astype(np.float64) * c
    off -= off.astype(np.float32).astype(np.float64)
    for lo, hi in ((120.0, 122.0), (122.0, 124.0), (124.0, 127.9), (-127.9, -124.0), (-124.0, -120.0)):
        pick = values[(off > lo) & (off < hi)][:4]
        assert len(pick)
        x = torch.from_numpy(pick)[:, None].expand(-1, vocab).contiguous()
        r = pkg.token_logprobs(x.to(dev), torch.zeros(len(pick), dtype=torch.int64, device=dev), entropy=True)
        ln = torch.full((len(pick),), math.log(vocab), dtype=torch.float64)
        # the exponent of up to 2^7 and log2 of the sum are off by 2 e of their size
        bound = 8 * 128 * E
        check(r.entropy, ln, bound, "entropy")
        check(r.logprobs, -ln, bound, "logprobs")
