"""Orthogonalised updates on the GPU against 64-bit Newton-Schulz steps: single elements to several tiles, odd sides, both
orientations, batches, every type.

Bounds, in the 2-norm over a matrix.  A step takes singular values through p(s) = a s + b s^3 + c s^5; as a map of
matrices it stretches a difference by at most L = max |p'|, |p(s) / s| over the values that occur, here 3.45.  A step's own error is
that of A, B and X as stored (22 bits: 2^-22 of them) and of fp32 sums of `side` or `other` terms, whose roundings are independent
(sqrt(terms) e), in the three products: at most 22 times their sum of the iterate's norm, as |a| + (|b| + 2 |c| s^2)
s^2 + ... is below 22 for s <= 1.2.  The iterate's norm is at most L^k after k steps from norm 1, and 1.2 sqrt(side).
Beside that bound the result is compared with the same steps in fp32 on the CPU, whose values have 24 bits: pairs,
with 22, are within eight times its error.  For a bf16 result the products' values have 11 bits, which the bound's worst case says
nothing about: there the same roundings are made in 64 bits, and the result is within twice their error, beside its own rounding;
that in turn is below 2^-9 of the norm."""
import math

import pytest
import torch

from test_gpu_step import E, TINY, UNIT, gen, types

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)
L = 3.45


def steps_of(x, steps=5, abc=ABC, eps=1e-7):
    """The definition, in x's own precision."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    a, b, c = abc
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def tolerance(rows, cols, steps):
    side, other = min(rows, cols), max(rows, cols)
    own = 22 * (2.0 ** -22 + 2 * math.sqrt(other) * E)
    return sum(L ** (steps - 1 - k) * own * min(L ** k, 1.2 * math.sqrt(side)) for k in range(steps))


def compare(got, want, rows, cols, steps=5, scale=1.0):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape and bool(got.isfinite().all())
    far = (got - want).norm(dim=(-2, -1))
    return far, tolerance(rows, cols, steps) * abs(scale)


def update(dtype, *shape):
    g = gen("ortho", *shape)
    rank = max(1, min(shape[-2:]) // 16)
    low = torch.randn(*shape[:-1], rank, generator=g) @ torch.randn(*shape[:-2], rank, shape[-1], generator=g)
    return ((low / math.sqrt(rank) + 0.2 * torch.randn(*shape, generator=g)) * 0.01).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (8, 8), (16, 40), (33, 31), (64, 64), (65, 130), (127, 128), (129, 64), (200, 333),
          (333, 200), (257, 256), (4, 500), (500, 4), (3, 5, 9), (5, 70, 66), (2, 3, 40, 100), (3, 150, 20)]


@types
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(pkg, dev, dtype, shape):
    x = update(dtype, *shape)
    want = steps_of(x.double())
    for out in {dtype, torch.float32}:
        got = pkg.orthogonalize(x.to(dev), dtype=out)
        assert got.dtype == out and got.shape == x.shape
        far, most = compare(got, want, *shape[-2:])
        norm = want.norm(dim=(-2, -1))
        assert bool((far <= most + 1.01 * UNIT[out] * norm + TINY[out]).all()), (far, most, norm)


@pytest.mark.parametrize("shape", [(64, 64), (200, 333), (333, 200), (2, 300, 260)], ids=str)
def test_as_good_as_single_precision(pkg, dev, shape):
    x = update(torch.float32, *shape)
    want = steps_of(x.double())
    far = (pkg.orthogonalize(x.to(dev)).double().cpu() - want).norm()
    single = (steps_of(x).double() - want).norm()
    assert float(far) <= 8 * float(single)


@pytest.mark.parametrize("width", [8, 136])
def test_each_element_of_22_bits(pkg, dev, width):
    """One step of c A A X on positive matrices of 8 x 8 (and zeros behind them), where nothing cancels: each element of
    the result has the relative errors of what it is made of.  X is in it five times, A twice, B once, each stored with 2^-22;
    four products leave out the product of the second parts, 2^-22 of them; and each of their sums of 8 terms rounds 8
    times, by at most a step, 2 E.  A stored element whose parts do not belong together would be 2^-11 off, an eighth of that here."""
    x = torch.zeros(4096, 8, width)
    x[:, :, :8] = 0.5 + torch.rand(4096, 8, 8, generator=gen("positive", width))
    want = steps_of(x.double(), steps=1, abc=(0.0, 0.0, 1.9))
    got = pkg.orthogonalize(x.to(dev), steps=1, coefficients=(0.0, 0.0, 1.9)).double().cpu()
    most = 12 * 2.0 ** -22 + 4 * 8 * 2 * E
    assert bool(((got - want).abs() <= most * want).all()), float(((got - want).abs() / want.clamp(min=1e-30)).max())


def half(x):
    """As stored for a product: times 2^12 in fp16."""
    return (x * 4096).half().double() / 4096


def fast_steps_of(x, steps=5):
    """The definition with the roundings of products of 11 bits."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.norm() + 1e-7)
    a, b, c = ABC
    for _ in range(steps):
        g = half(half(x) @ half(x).mT)
        poly = half(b * g + c * (g @ g))
        x = a * x + poly @ half(x)
    return x.mT if tall else x


@pytest.mark.parametrize("shape", [(64, 64), (200, 333), (520, 300), (768, 700)], ids=str)
def test_products_of_11_bits(pkg, dev, shape):
    x = update(torch.float32, *shape)
    want = steps_of(x.double())
    norm = float(want.norm())
    emulated = float((fast_steps_of(x.double()) - want).norm())
    assert emulated < norm * 2.0 ** -9
    far = float((pkg.orthogonalize(x.to(dev), dtype=torch.bfloat16).double().cpu() - want).norm())
    # in the mean square a rounding is off by 1 / sqrt(3) of its bound at most
    assert far <= 2 * emulated + UNIT[torch.bfloat16] * norm * 0.6, (far / norm, emulated / norm)


@pytest.mark.parametrize("shape", [(2, 1030, 1100), (1100, 520), (40, 300, 280)], ids=str)
def test_large_tiles(pkg, dev, shape):
    x = update(torch.bfloat16, *shape).to(dev)
    want = steps_of(x.double()).cpu()
    got = pkg.orthogonalize(x, dtype=torch.float32)
    far, most = compare(got, want, *shape[-2:])
    assert bool((far <= most + 1.01 * UNIT[torch.float32] * want.norm(dim=(-2, -1))).all())


@types
def test_base_scale_and_place(pkg, dev, dtype):
    x = update(torch.bfloat16, 3, 50, 90)
    base = torch.randn(3, 50, 90, generator=gen("base")).to(dtype)
    ortho = steps_of(x.double())
    want = 0.9 * base.double() - 0.3 * ortho
    most = (0.3 * tolerance(50, 90, 5) + (UNIT[dtype] * 1.01 + 4 * E) * (want.norm() + base.double().norm() * E)
            + TINY[dtype] * want.numel())
    weight = base.to(dev)
    got = pkg.orthogonalize(x.to(dev), scale=-0.3, base=weight, keep=0.9)
    assert got.dtype == dtype and torch.equal(weight.cpu(), base)
    assert float((got.double().cpu() - want).norm()) <= float(most) * math.sqrt(3)
    version = weight._version
    again = pkg.orthogonalize(x.to(dev), scale=-0.3, base=weight, keep=0.9, out=weight)
    assert again.data_ptr() == weight.data_ptr() and weight._version > version and torch.equal(weight, got)
    over = x.to(dev).clone()
    assert torch.equal(pkg.orthogonalize(over, out=over), pkg.orthogonalize(x.to(dev)))


def test_strided_rows(pkg, dev):
    wide = torch.full((70, 200), 3.0, device=dev)
    x = update(torch.float32, 70, 90).to(dev)
    want = pkg.orthogonalize(x)
    for lo in (0, 1, 50):
        view = wide[:, lo:lo + 90]
        view.copy_(x)
        out = torch.full((70, 101), 5.0, device=dev)
        far = (pkg.orthogonalize(view, out=out[:, 3:93]) - want).norm()
        # the squares are added in another order: one rounding of |x|
        assert float(far) <= 1e-4 * float(want.norm())
        assert bool((out[:, :3] == 5).all()) and bool((out[:, 93:] == 5).all())


@pytest.mark.parametrize("steps,abc", [(1, ABC), (2, (2.0, -1.5, 0.5)), (12, (1.5, -0.5, 0.0)), (10, ABC)])
def test_steps_and_coefficients(pkg, dev, steps, abc):
    x = update(torch.float32, 60, 100)
    want = steps_of(x.double(), steps, abc)
    got = pkg.orthogonalize(x.to(dev), steps=steps, coefficients=abc).double().cpu()
    stretch = max(1.0, min(L, abc[0])) ** min(steps, 5)   # what has grown to the values near 1 grows no more
    assert float((got - want).norm()) <= steps * 22 * stretch * (2.0 ** -22 + 20 * E) * 1.2 * math.sqrt(60)


@pytest.mark.parametrize("cols", [100, 200])
@pytest.mark.parametrize("least", [1e-36, -1e-30, 1e-20])
def test_next_to_no_fifth_powers(pkg, dev, cols, least):
    """A coefficient that is rounded off is as good as none: b over it is never taken."""
    x = update(torch.float32, 60, cols).to(dev)
    assert torch.equal(pkg.orthogonalize(x, coefficients=(1.5, -0.5, least)), pkg.orthogonalize(x, coefficients=(1.5, -0.5, 0.0)))


def test_singular_values_go_towards_one(pkg, dev):
    x = torch.randn(128, 256, generator=gen("spread")).to(dev)
    s = torch.linalg.svdvals(pkg.orthogonalize(x).double())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.25


def test_zeros_and_unsound_matrices_stay_alone(pkg, dev):
    x = update(torch.float32, 5, 40, 72)
    x[1] = 0
    x[3, 20, 5] = math.nan
    x[4, 0, 0] = math.inf
    got = pkg.orthogonalize(x.to(dev)).cpu()
    assert not got[1].any() and got[3].isnan().all() and got[4].isnan().all()
    for i in (0, 2):
        assert torch.equal(got[i], pkg.orthogonalize(x[i].to(dev)).cpu())
    base = torch.ones(40, 72, device=dev)
    assert bool((pkg.orthogonalize(x[1].to(dev), base=base, keep=0.5) == 0.5).all())


@types
def test_any_magnitude(pkg, dev, dtype):
    """|x| may be near the type's ends; only eps is a scale."""
    x = torch.randn(30, 50, generator=gen("magnitude"))
    for power in (-10, -4, 0, 2 if dtype == torch.float16 else 30):
        y = (x * 10.0 ** power).to(dtype)
        want = steps_of(y.double())
        far, most = compare(pkg.orthogonalize(y.to(dev), dtype=torch.float32), want, 30, 50)
        assert float(far) <= most + 4 * UNIT[torch.float32] * float(want.norm()), power


def test_none(pkg, dev):
    assert pkg.orthogonalize(torch.empty(0, 4, 6, device=dev)).shape == (0, 4, 6)


def test_refusals(pkg, dev):
    x = torch.randn(8, 12, device=dev)
    for call, what in (
            (lambda: pkg.orthogonalize(x, steps=0), "steps"), (lambda: pkg.orthogonalize(x, steps=65), "steps"),
            (lambda: pkg.orthogonalize(x, coefficients=(1.0, 2.0)), "unpack"),
            (lambda: pkg.orthogonalize(x, coefficients=(1.0, 2.0, 2e3)), "1024"),
            (lambda: pkg.orthogonalize(x, eps=0.0), "eps"), (lambda: pkg.orthogonalize(x, scale=math.nan), "finite"),
            (lambda: pkg.orthogonalize(x, dtype=torch.float64), "dtype"),
            (lambda: pkg.orthogonalize(x, dtype=torch.float16, out=x.clone()), "out is"),
            (lambda: pkg.orthogonalize(x, base=x.half(), out=x.clone()), "base must be"),
            (lambda: pkg.orthogonalize(x, base=x[:, :5]), "shape"),
            (lambda: pkg.orthogonalize(x[0]), "two dimensions"),
            (lambda: pkg.orthogonalize(x[:0]), "at least one row"),
            (lambda: pkg.orthogonalize(x.t()), "adjacent"),
            (lambda: pkg.orthogonalize(x.view(2, 4, 12)[:, :2]), "adjacent"),
            (lambda: pkg.orthogonalize(x.view(-1)[:48].view(4, 12), out=x.view(-1)[12:60].view(4, 12)), "shares"),
            (lambda: pkg.orthogonalize(x.double()), "float32, bfloat16")):
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(pkg.ECError):
        pkg.orthogonalize(torch.empty(1, 65537, device=dev))
