"""The log probabilities' entropy and gradient where logits are large: finite masks, dominating logits, rows
masked throughout.  Bounds as in test_gpu_step.py."""
import math

import numpy as np
import pytest
import torch

from test_gpu_step import E, TINY, UNIT, check, gen, logp_bounds, logp_want, types

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


# ---------------------------------------------------------------- gradient --

def formula(x, target, scale, lse, ent, g, h):
    """The gradient in 64 bits from the given lse and entropy, p at most 1, and the bound of its evaluation in fp32: scale x
    is rounded (nothing at scale 1), the difference to lse and its product with log2 e are each off by e of
    their size, and log2 e, exp2 and the other factors by less than 8 e."""
    z = x.double() * float(np.float32(scale))                # as the operator is given it
    d = (z - lse.double()[:, None]).clamp(max=0)
    p = d.exp()
    ok = (target >= 0) & (target < x.shape[1])
    g = torch.where(ok, g.double(), 0.0)[:, None]
    h, ent = h.double()[:, None], ent.double()[:, None]
    d = torch.where(p > 0, d, 0.0)
    z = torch.where(p > 0, z, 0.0)
    exponent = (z.abs() if scale != 1 else 0.0) + 4 * d.abs() + 8
    hot = torch.zeros_like(z).scatter_(1, torch.where(ok, target, 0)[:, None], g)
    want = (hot - p * (g + h * (d + ent))) * scale
    by = g.abs() + h.abs() * (d.abs() + ent.abs())
    more = (p * (by * exponent + h.abs() * exponent) + hot.abs() * 4) * E * scale + 2.0 ** -120
    return want, more


@pytest.mark.parametrize("scale", [1.0, 1.3], ids=["1", "1.3"])
@pytest.mark.parametrize("shift", [0.0, 100.0, -1000.0, 20_000.0])
def test_grad_follows_the_given_lse(pkg, dev, shift, scale):
    """Logits far from zero: the exponent is as exact as the log of the sum that it is given."""
    g = gen("shifted", shift)
    rows, vocab = 4, 32_063
    x = torch.randn(rows, vocab, generator=g) * 3 + shift
    x[:, 17] = -math.inf
    target = torch.tensor([3, -100, vocab - 1, 40])
    dlp, dent = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    r = pkg.token_logprobs(x.to(dev), target.to(dev), scale=scale, entropy=True)
    for h in (dent, torch.zeros(rows)):
        want, more = formula(x, target, scale, r.lse.cpu(), r.entropy.cpu(), dlp, h)
        kw = dict(entropy=r.entropy, dentropy=h.to(dev)) if h is dent else {}
        got = pkg.token_logprobs_grad(x.to(dev), target.to(dev), r.lse, dlp.to(dev), scale=scale, **kw)
        check(got, want, rounded(want, more), f"shift {shift}")


def rounded(want, more, dtype=torch.float32):
    return want.abs() * UNIT[dtype] * 1.01 + TINY[dtype] + more * 1.01


@types
@pytest.mark.parametrize("scale", [1.0, 1 / 0.6, 0.3], ids=["1", "1.67", "0.3"])
def test_grad_of_a_dominating_logit(pkg, dev, dtype, scale):
    """One logit far above the others has probability 1, whatever its size: no gradient where it is the target, and
    minus the others' where it is not."""
    sizes = [50.0, 1e3, 65504.0, 1e6, 1e8, 1e9, 3.3e20, 1e38, 2e38]
    sizes += [-s for s in sizes]
    sizes = [s for s in sizes if abs(s) <= torch.finfo(dtype).max]
    vocab = 1003
    x = torch.full((len(sizes), vocab), -math.inf, dtype=dtype)
    x[:, 5] = torch.tensor(sizes, dtype=dtype)
    for i, s in enumerate(sizes):
        if s > 0:
            x[i, 100:] = -s / 2 if s > 1e4 else -60.0
            x[i, 200:] = 0.0 if s > 1e4 else -70.0
    target = torch.full((len(sizes),), 5, device=dev)
    ones = torch.ones(len(sizes), device=dev)
    r = pkg.token_logprobs(x.to(dev), target, scale=scale, entropy=True)
    dominates = x[:, 5].float() * scale                      # rounded as the kernels round it
    assert torch.equal(r.lse.cpu(), dominates)
    # relative to a reference that is off by e of itself, past 2^7 of which the row is gone over again
    near = 4 * E * (1 + (dominates.abs() * 1.45 * E).clamp(max=128))
    check(r.logprobs, near * 0, near, "logprobs")
    check(r.entropy, near * 0, near * 2, "entropy")
    for kw in ({}, dict(entropy=r.entropy, dentropy=ones)):
        got = pkg.token_logprobs_grad(x.to(dev), target, r.lse, ones, scale=scale, **kw)
        # g - p (g + h H) with p = 1, the sum in brackets rounded; H is what the forward pass gave, 0 but for `near`
        check(got[:, 5], near * 0, (r.entropy.cpu().abs() * 1.01 + 2 * E) * scale + TINY[dtype] if kw else 0.0, "at the target")
        h = ones.cpu() * len(kw) / 2
        want, more = formula(x, target.cpu(), scale, r.lse.cpu(), r.entropy.cpu(), ones.cpu(), h)
        check(got[:, 6:], want[:, 6:], rounded(want, more, dtype)[:, 6:], "beside it")
        assert not bool(got[:, :5].any())
        # the target elsewhere: all of the gradient goes through the dominating logit, but for rows that count as masked
        other = pkg.token_logprobs_grad(x.to(dev), target - 5, r.lse, ones, scale=scale, **kw).cpu().float()
        want = torch.tensor(0.0)
        for i, s in enumerate(sizes):
            masked = float(x[i, 5]) * scale < -2.0 ** 127 / math.log2(math.e) * min(1.0, scale)
            want = 0.0 if masked else scale
            assert abs(float(other[i, 0]) - want) <= scale * (UNIT[dtype] + 4 * E) + TINY[dtype]
            entropy = float(r.entropy[i].abs()) * scale if kw else 0.0
            assert abs(float(other[i, 5]) + want) <= scale * (UNIT[dtype] + 4 * E) + TINY[dtype] + entropy * 1.01


@types
@pytest.mark.parametrize("scale", [1.0, 1 / 0.6, 0.3], ids=["1", "1.67", "0.3"])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e10, -1e30, "half", "lowest"])
def test_grad_of_rows_masked_throughout(pkg, dev, dtype, mask, scale):
    """A row of one finite value: probabilities from the lse it has in fp32, never above 1; nothing where that is below
    the masks' bound, nor at an ignored position without an entropy's gradient."""
    vocab = 1000
    low = torch.finfo(dtype).min
    value = low if mask == "lowest" else low / 2 if mask == "half" else mask
    if value < low:
        pytest.skip("not of this type")
    x = torch.full((2, vocab), value).to(dtype)
    target = torch.tensor([5, -100])
    ones = torch.ones(2)
    r = pkg.token_logprobs(x.to(dev), target.to(dev), scale=scale, entropy=True)
    z = float(x[0, 0]) * scale
    lse = r.lse.cpu().double()
    assert bool(((lse - z).abs() <= abs(z) * 3 * E + 7).all() | (lse == -math.inf).all())
    masked = z < -2.0 ** 127 / math.log2(math.e) * min(1.0, scale)
    for kw in ({}, dict(entropy=r.entropy, dentropy=ones.to(dev))):
        got = pkg.token_logprobs_grad(x.to(dev), target.to(dev), r.lse, ones.to(dev), scale=scale, **kw).cpu()
        assert bool(got.isfinite().all())
        if not kw:
            assert not bool(got[1].any())
        if masked:
            assert not bool(got.any())
            continue
        # the exponent is the fp32 difference of the rounded product and lse
        d = torch.clamp(x.float() * scale - r.lse.cpu()[:, None], max=0).double()
        p = d.exp()
        g = torch.tensor([[1.0], [0.0]], dtype=torch.float64)
        h = 1.0 if kw else 0.0
        inner = d + r.entropy.cpu().double()[:, None]
        hot = torch.zeros(2, vocab, dtype=torch.float64)
        hot[0, 5] = 1.0
        want = (hot - p * (g + h * inner)) * scale
        more = (p * (g + h * (inner.abs() + 1)) * (4 * d.abs() + 8) + hot * 4 + p * h * 16) * E * scale
        check(got, want, rounded(want, more, dtype), f"mask {mask}")


@types
def test_grad_of_unsound_rows(pkg, dev, dtype):
    """NaN and +infinity stay visible: all of their row's gradient by the lse of the forward pass, their own by a finite one."""
    x = torch.randn(3, 70, generator=gen("unsound")).to(dtype)
    x[0, 9], x[1, 69], x[2, 3] = math.nan, math.inf, -math.inf
    target = torch.tensor([1, 2, 4], device=dev)
    ones = torch.ones(3, device=dev)
    r = pkg.token_logprobs(x.to(dev), target, entropy=True)
    for kw in ({}, dict(entropy=r.entropy, dentropy=ones)):
        got = pkg.token_logprobs_grad(x.to(dev), target, r.lse, ones, **kw).cpu()
        assert bool(got[:2].isnan().all()) and bool(got[2].isfinite().all()) and got[2, 3] == 0
    got = pkg.token_logprobs_grad(x.to(dev), target, ones * 5, ones).cpu()
    assert got.isnan().nonzero().tolist() == [[0, 9]] and bool(got.nan_to_num().isfinite().all())
