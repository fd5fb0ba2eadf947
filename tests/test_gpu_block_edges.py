"""The block operators' edges on the GPU: empty batches, iterates that grow, tangents, longest rows."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import test_gpu_block_norms as norms
from test_gpu_block_ortho import steps_of, update
from test_gpu_step import E, UNIT, check, gen, rounded, types

pytestmark = pytest.mark.gpu


@types
@pytest.mark.parametrize("width,inner", [(2048, 1000), (256, 256), (64, 512), (65, 4001)])
def test_gated_ff_grad_without_rows(pkg, dev, dtype, width, inner):
    """An empty batch, as an expert without tokens has it, at widths whose sums are split along k with rows."""
    w = torch.randn(2 * inner, width, device=dev).to(dtype)
    x, dh = (torch.empty(0, v, dtype=dtype, device=dev) for v in (width, inner))
    for out in {dtype, torch.float32}:
        got = pkg.gated_ff_grad(dh, x, w[:inner], w[inner:], dtype=out)
        assert got.dx.shape == (0, width) and not got.dw_gate.any() and not got.dw_up.any()
    into = [torch.ones(inner, width, device=dev) for _ in range(2)]
    pkg.gated_ff_grad(dh, x, w[:inner], w[inner:], out=into, accumulate=True)
    assert all(bool((t == 1).all()) for t in into)
    leaves = [x.requires_grad_(), w[:inner].clone().requires_grad_(), w[inner:].clone().requires_grad_()]
    pkg.gated_ff(*leaves).sum().backward()
    assert leaves[0].grad.shape == (0, width) and not any(bool(t.grad.any()) for t in leaves[1:])


@types
def test_the_input_gradient_of_no_rows(pkg, dev, dtype):
    """Of an empty batch with frozen weights: an empty dx, alone and through autograd."""
    w = torch.randn(600, 512, device=dev).to(dtype)
    for lead in ((0,), (3, 0)):
        x, dh = (torch.empty(*lead, v, dtype=dtype, device=dev) for v in (512, 300))
        got = pkg.gated_ff_grad(dh, x, w[:300], w[300:], weights=False)
        assert got.dx.shape == x.shape and got.dw_gate is None and got.dw_up is None
        got = pkg.gated_ff_grad(dh, x, w[:300], w[300:], inputs=False)
        assert got.dx is None and not got.dw_gate.any() and not got.dw_up.any()
        pkg.gated_ff(x.requires_grad_(), w[:300], w[300:]).sum().backward()
        assert x.grad.shape == x.shape


def grown(s, abc, steps):
    """Singular values from s on, step by step."""
    a, b, c = abc
    values = [s]
    for _ in range(steps):
        s = values[-1]
        values.append(a * s + b * s ** 3 + c * s ** 5)
    return values


def nearly_one(rows, cols):
    """A matrix whose largest singular value is close to its norm."""
    g = gen("grown", rows, cols)
    u, v = (torch.randn(k, 1, generator=g, dtype=torch.float64) for k in (rows, cols))
    x = u @ v.T + 0.02 * torch.randn(rows, cols, generator=g, dtype=torch.float64)
    return (x / x.norm()).float()


GROWING = [((4.0, 0.0, 0.0), 2), ((4.0, 0.0, 0.0), 9), ((0.0, 0.0, 3.0), 3), ((2.5, 1.0, 0.5), 3), ((1.5, 1.5, 0.0), 4),
           ((14.9, 0.0, 0.0), 2), ((1024.0, 0.0, 0.0), 3), ((0.01, 0.0, 0.0), 5), ((0.001, 0.0005, 0.0), 4), ((30.0, 20.0, 10.0), 2), ((0.0, 1024.0, 0.0), 2), ((0.0, 0.0, 1024.0), 2)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (60, 100), (100, 60), (150, 200), (200, 150), (300, 520)], ids=str)
def test_growing_iterates(pkg, dev, shape, out):
    """Coefficients that take singular values far from 1, to 2^20 or 2^-30 before the last step.

    With a, b, c >= 0 a step p stretches a difference by at most p'(s) at the largest singular value s, and s p' <= 5 p: errors
    relative to it grow by 5 a step at most.  A step's own, relative to p(s) and over `side` singular values: X is in it five times,
    A twice, B once as stored, and so are the products' left out second parts, and four sums of `other` terms, whose
    roundings by at most 2 E are independent.  X as stored has 22 bits, or 11 for a bf16 result of 64 rows and more."""
    x = nearly_one(*shape)
    side, other = min(shape), max(shape)
    bits = 11 if out == torch.bfloat16 and side >= 64 else 22
    own = 12 * 2.0 ** -bits + 4 * 2 * E * math.sqrt(other)
    for abc, steps in GROWING:
        want = steps_of(x.double(), steps, abc)
        most = grown(float(torch.linalg.matrix_norm(x.double(), 2)), abc, steps)[-1]
        got = pkg.orthogonalize(x.to(dev), steps=steps, coefficients=abc, dtype=out).double().cpu()
        assert bool(got.isfinite().all()), (abc, steps)
        bound = most * math.sqrt(side) * own * sum(5.0 ** k for k in range(steps)) + 1.01 * UNIT[out] * float(want.norm())
        assert float((got - want).norm()) <= bound, (abc, steps, float((got - want).norm()) / most)


@pytest.mark.parametrize("shape", [(1, 1), (60, 100), (150, 200)], ids=str)
def test_iterates_past_the_range_are_not_finite(pkg, dev, shape):
    """2^30 before the last step: past 2^20, and said by what comes out."""
    got = pkg.orthogonalize(nearly_one(*shape).to(dev), steps=4, coefficients=(1024.0, 0.0, 0.0))
    assert not bool(got.isfinite().all())


def test_tangents_are_refused(pkg, dev):
    """A tangent of any operand, and what torch's own transforms make of one."""
    one, v = torch.ones(8, 8, device=dev), torch.ones(8, device=dev)
    tokens = torch.zeros(8, dtype=torch.int64, device=dev)
    calls = {"x": lambda t: pkg.gated_ff(t, one, one), "w_up": lambda t: pkg.gated_ff(one, one, t),
             "dh": lambda t: pkg.gated_ff_grad(t, one, one, one), "branch": lambda t: pkg.residual_norm(one, t, weight=v),
             "weight": lambda t: pkg.residual_norm(one, weight=t[0].clone()), "gate": lambda t: pkg.residual_norm(one, one, gate=t),
             "dresidual": lambda t: pkg.residual_norm_grad(t, None, one, one), "base": lambda t: pkg.orthogonalize(one, base=t),
             "table": lambda t: pkg.embed(tokens, t), "logits": lambda t: pkg.token_logprobs(t, tokens),
             "dout": lambda t: pkg.embed_grad(tokens, t, 8)}
    for name, call in calls.items():
        with forward_ad.dual_level(), pytest.raises(ValueError, match=f"{name} has a forward-mode tangent"):
            call(forward_ad.make_dual(one, one))
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (one,), (one,))
        call(one)
    leaf = one.clone().requires_grad_()
    with forward_ad.dual_level(), pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        pkg.gated_ff(forward_ad.make_dual(leaf, one), one, one)


def test_a_pair_in_one_tensor(pkg, dev):
    """The weights' gradients into the halves of one tensor [2, inner, width], given as it is."""
    x, w, dh = (torch.randn(*s, device=dev) for s in ((40, 24), (32, 24), (40, 16)))
    want = pkg.gated_ff_grad(dh, x, w[:16], w[16:])
    out = torch.empty(2, 16, 24, device=dev)
    pkg.gated_ff_grad(dh, x, w[:16], w[16:], dtype=torch.float32, out=out)
    assert torch.equal(out[0], want.dw_gate) and torch.equal(out[1], want.dw_up)


@pytest.mark.parametrize("dtype,n,width,gates", [
    (torch.float32, 301, 9001, 1), (torch.float32, 600, 8200, 300), (torch.float32, 603, 16384, 603),
    (torch.bfloat16, 1301, 9001, 1), (torch.bfloat16, 600, 8200, 300), (torch.float16, 603, 16384, 603),
    (torch.float16, 1800, 8203, 600), (torch.float32, 1100, 8193, 4)], ids=str)
def test_longest_rows(pkg, dev, dtype, n, width, gates):
    """Rows whose sums over rows are partly in LDS, for teams of several rows: parts of a gate's rows, and whole gates, whose
    sums are written and begun anew row by row of the gate."""
    o = norms.operands(dtype, n, width, gates, True, True)
    o = {k: v.to(dev) for k, v in o.items()}
    rest = {k: o[k] for k in ("gate", "branch_weight", "weight")}
    r = pkg.residual_norm(o["residual"], o["branch"], scale=0.4, **rest)
    for name, (value, bound) in norms.forward(o, 0.4).items():
        check(getattr(r, name), value, rounded(value, getattr(r, name).dtype, bound).cpu(), name)
    g = gen("dlongest", n, width)
    ds, dn = (torch.randn(n, width, generator=g).to(dtype).to(dev) for _ in range(2))
    saved = dict(rstd=r.rstd, branch_rstd=r.branch_rstd, scale=0.4, **rest)
    got = pkg.residual_norm_grad(ds, dn, r.residual, o["branch"], **saved)
    for name, (value, bound) in norms.gradients(o, r.residual, ds, dn, r.rstd, r.branch_rstd, 0.4).items():
        v = getattr(got, name)
        check(v, value, rounded(value, v.dtype, bound * 1.05).cpu(), name)
    again = pkg.residual_norm_grad(ds, dn, r.residual, o["branch"], **saved)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("n", [5, 300])
def test_fp16_gradients_past_the_type_are_not_finite(pkg, dev, n):
    """dg = dh u act' past 65504 is infinite, as any fp16 gradient, and shows in every result that it is part of; the rows and
    outputs beside it stay."""
    g = gen("overflow", n)
    x = torch.randn(n, 64, generator=g).half()
    w = (torch.randn(96, 64, generator=g) / 80).half()
    dh = torch.randn(n, 48, generator=g).half()
    x[2] = 4.0
    w[48 + 7], w[7] = 1.0, 0.01   # u = 256, g = 2.56 of row 2, output 7
    dh[2, 7] = 6e4
    got = pkg.gated_ff_grad(dh.to(dev), x.to(dev), w[:48].to(dev), w[48:].to(dev), dtype=torch.float32)
    assert not got.dx[2].isfinite().any() and not got.dw_gate[7].isfinite().any()
    rows, outputs = [i for i in range(n) if i != 2], [i for i in range(48) if i != 7]
    assert bool(got.dx[rows].isfinite().all())
    assert bool(got.dw_gate[outputs].isfinite().all()) and bool(got.dw_up[outputs].isfinite().all())


@pytest.mark.parametrize("out", [torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(128, 128), (100, 60), (60, 100), (127, 65), (64, 64), (300, 90), (129, 200)], ids=str)
def test_small_updates_keep_22_bits(pkg, dev, shape, out):
    """Within eight times the error of the same steps in fp32, whose values have 24 bits, by rows and columns too (against the largest
    one's); products of 11 bits are a hundred times that.  A result's own rounding has a mean square of a third of its
    bound's, and over a row's values not above it."""
    x = update(torch.float32, *shape)
    want = steps_of(x.double())
    near = steps_of(x).double() - want
    far = pkg.orthogonalize(x.to(dev), dtype=out).double().cpu() - want
    assert float(far.norm()) <= 8 * float(near.norm()) + 0.6 * UNIT[out] * float(want.norm())
    for d in (0, 1):
        assert bool((far.norm(dim=d) <= 8 * near.norm(dim=d).max() + UNIT[out] * 1.01 * want.norm(dim=d)).all()), d
