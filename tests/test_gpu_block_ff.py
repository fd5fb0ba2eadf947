"""The gated feed-forward and its gradients on the GPU against 64-bit products: one row to many, odd widths, strides
and addresses, every type and activation.

Bounds.  With |x| |w| the product of magnitudes, an fp32 sum of n terms on the matrix cores is off by at most 2 n e
of its sum of magnitudes (e = 2^-24; the cores may truncate where they add, hence twice).  Activations and their derivatives are
taken as 32 e off relative to |g| + 1, which covers the exponential's argument; their slopes are at most 1.13, their
second derivatives at most 1."""
import math

import pytest
import torch

from test_gpu_step import E, UNIT, check, gen, rounded, types

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh"]
SLOPE, BEND = 1.13, 1.0


def activate(g, act):
    """The activation and its derivative in 64 bits."""
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    z, dz = g, torch.ones_like(g)
    if act == "gelu_tanh":
        z = math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3)
        dz = math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(z)
    return g * s, s + g * s * (1 - s) * dz


def forward(x, wg, wu, act):
    """h, and the bound of its fp32 value before the rounding."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.T, x @ wu.T
    off = 2 * (x.shape[1] + 2) * E
    dg, du = off * (x.abs() @ wg.abs().T), off * (x.abs() @ wu.abs().T)
    a, slope = activate(g, act)
    da = SLOPE * dg + 32 * E * (g.abs() + 1)
    return a * u, da * (u.abs() + du) + a.abs() * du, (g, u, dg, du, a, slope, da)


def gradients(dh, x, wg, wu, act, dtype, out):
    """dx, dw_gate, dw_up and their bounds."""
    _, _, (g, u, eg, eu, a, slope, ea) = forward(x, wg, wu, act)
    dh, x, wg, wu = dh.double(), x.double(), wg.double(), wu.double()
    n, f = dh.shape
    eslope = BEND * eg + 32 * E * (g.abs() + 1)
    dg, du = dh * u * slope, dh * a
    bg = dh.abs() * (eu * (slope.abs() + eslope) + u.abs() * eslope) + 4 * E * dg.abs()
    bu = dh.abs() * ea + 4 * E * du.abs()
    # what the products read is rounded: once, or with few rows to two parts
    part = UNIT[dtype] if dtype == torch.float32 or n > 256 else UNIT[dtype] ** 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bg, bu = bg + part * 1.01 * dg.abs() + tiny, bu + part * 1.01 * du.abs() + tiny
    results = []
    for want, bound, terms, kind in (
            (dg @ wg + du @ wu, bg @ wg.abs() + bu @ wu.abs(), 4 * f, dtype),
            (dg.T @ x, bg.T @ x.abs(), 2 * n, out), (du.T @ x, bu.T @ x.abs(), 2 * n, out)):
        sums = dg.abs() @ wg.abs() + du.abs() @ wu.abs() if not results else \
            (dg if len(results) == 1 else du).abs().T @ x.abs()
        results.append((want, rounded(want, kind, bound + 2 * (terms + 4) * E * (sums + bound))))
    return results


def operands(dtype, n, width, inner, key=0):
    g = gen("ff", n, width, inner, key)
    x = torch.randn(n, width, generator=g).to(dtype)
    w = (torch.randn(2 * inner, width, generator=g) / math.sqrt(width)).to(dtype)
    return x, w, (torch.randn(n, inner, generator=g) * 0.1).to(dtype)


SIZES = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (17, 64, 96), (64, 72, 129), (65, 127, 33), (129, 200, 257), (300, 65, 520),
         (1, 2048, 515), (256, 136, 72), (257, 264, 264), (1000, 40, 24)]
sizes = pytest.mark.parametrize("n,width,inner", SIZES, ids=lambda v: str(v))


@types
@sizes
def test_gated_ff(pkg, dev, dtype, n, width, inner):
    x, w, _ = operands(dtype, n, width, inner)
    act = ACTS[(n + width) % 3]
    want, bound, _ = forward(x, w[:inner], w[inner:], act)
    w = w.to(dev)
    got = pkg.gated_ff(x.to(dev), w[:inner], w[inner:], activation=act)
    assert got.dtype == dtype and got.shape == (n, inner)
    check(got, want, rounded(want, dtype, bound), "h")


@types
@sizes
def test_gated_ff_grad(pkg, dev, dtype, n, width, inner):
    x, w, dh = operands(dtype, n, width, inner)
    act = ACTS[(n + inner) % 3]
    wd = w.to(dev)
    for out in {dtype, torch.float32}:
        got = pkg.gated_ff_grad(dh.to(dev), x.to(dev), wd[:inner], wd[inner:], activation=act, dtype=out)
        assert got.dx.dtype == dtype and got.dw_gate.dtype == got.dw_up.dtype == out
        for name, g, (want, bound) in zip(got._fields, got, gradients(dh, x, w[:inner], w[inner:], act, dtype, out)):
            check(g, want, bound, name)


@types
def test_large_tiles(pkg, dev, dtype):
    """Enough tiles that the large ones are taken, with ends in both directions."""
    n, width, inner = (4100, 136, 4100) if dtype != torch.float32 else (4100, 68, 4100)
    x, w, dh = (t.to(dev) for t in operands(dtype, n, width, inner))
    want, bound, _ = forward(x, w[:inner], w[inner:], "silu")
    check(pkg.gated_ff(x, w[:inner], w[inner:]), want, rounded(want, dtype, bound).cpu(), "h")
    got = pkg.gated_ff_grad(dh, x, w[:inner], w[inner:])
    for name, g, (want, bound) in zip(got._fields, got, gradients(dh, x, w[:inner], w[inner:], "silu", dtype, dtype)):
        check(g, want, bound.cpu(), name)


@types
@pytest.mark.parametrize("n", [40, 300])
def test_strides_and_addresses(pkg, dev, dtype, n):
    """Rows of wider buffers at any element, and results within wider buffers whose other elements stay."""
    width, inner = 96, 80
    x, w, dh = operands(dtype, n, width, inner)
    want, bound, _ = forward(x, w[:inner], w[inner:], "gelu")
    for lo, pad in ((0, 32), (1, 15), (8, 40), (3, 5)):
        def inside(t):
            buffer = torch.full((t.shape[0], t.shape[1] + pad), 7.0, dtype=t.dtype, device=dev)
            view = buffer[:, lo:lo + t.shape[1]] if lo + t.shape[1] <= buffer.shape[1] else buffer[:, :t.shape[1]]
            view.copy_(t)
            return buffer, view
        (_, xs), (_, gs), (_, us), (_, ds) = (inside(t) for t in (x, w[:inner], w[inner:], dh))
        buffer, out = inside(torch.zeros(n, inner, dtype=dtype))
        assert pkg.gated_ff(xs, gs, us, activation="gelu", out=out) is not None
        check(out, want, rounded(want, dtype, bound), "h")
        assert int((buffer == 7.0).sum()) >= n * pad
        pair = [inside(torch.ones(inner, width))for _ in range(2)]
        got = pkg.gated_ff_grad(ds, xs, gs, us, activation="gelu", out=[v for _, v in pair], accumulate=True)
        wants = gradients(dh, x, w[:inner], w[inner:], "gelu", dtype, torch.float32)
        check(got.dx, *wants[0], "dx")
        for (b, v), (want_w, bound_w) in zip(pair, wants[1:]):
            check(v, want_w + 1.0, bound_w + 2 * E * (want_w.abs() + 1.0), "dw added to ones")
            assert int((b == 7.0).sum()) >= inner * pad


@types
@pytest.mark.parametrize("n", [7, 90, 300])
def test_weights_of_different_strides(pkg, dev, dtype, n):
    """Each weight with rows as far apart as its own buffer has them, one of them perhaps not to be read in place."""
    width, inner = 64, 72
    x, w, dh = operands(dtype, n, width, inner)
    want, bound, _ = forward(x, w[:inner], w[inner:], "silu")
    wants = gradients(dh, x, w[:inner], w[inner:], "silu", dtype, dtype)
    for gate_pad, up_pad in ((0, 64), (192, 0), (8, 16), (0, 1), (3, 0)):
        views = []
        for t, pad in ((w[:inner], gate_pad), (w[inner:], up_pad)):
            views.append(torch.full((inner, width + pad), 9.0, dtype=dtype, device=dev)[:, :width])
            views[-1].copy_(t)
        check(pkg.gated_ff(x.to(dev), *views), want, rounded(want, dtype, bound), "h")
        got = pkg.gated_ff_grad(dh.to(dev), x.to(dev), *views)
        for name, g, (value, most) in zip(got._fields, got, wants):
            check(g, value, most, name)


def test_leading_dimensions_and_one_side(pkg, dev):
    x, w, dh = (t.to(dev) for t in operands(torch.bfloat16, 6 * 5, 32, 48))
    g, u = w[:48], w[48:]
    h = pkg.gated_ff(x.view(6, 5, 32), g, u)
    assert h.shape == (6, 5, 48) and torch.equal(h.view(30, 48), pkg.gated_ff(x, g, u))
    both = pkg.gated_ff_grad(dh.view(6, 5, 48), x.view(6, 5, 32), g, u)
    assert both.dx.shape == (6, 5, 32)
    only = pkg.gated_ff_grad(dh, x, g, u, weights=False)
    assert only.dw_gate is None and only.dw_up is None and torch.equal(only.dx, both.dx.view(30, 32))
    only = pkg.gated_ff_grad(dh, x, g, u, inputs=False)
    assert only.dx is None and torch.equal(only.dw_gate, both.dw_gate) and torch.equal(only.dw_up, both.dw_up)


def test_no_rows(pkg, dev):
    w = torch.randn(20, 16, device=dev)
    x, dh = torch.empty(0, 16, device=dev), torch.empty(0, 10, device=dev)
    assert pkg.gated_ff(x, w[:10], w[10:]).shape == (0, 10)
    got = pkg.gated_ff_grad(dh, x, w[:10], w[10:])
    assert got.dx.shape == (0, 16) and not got.dw_gate.any() and not got.dw_up.any()
    kept = [torch.ones(10, 16, device=dev) for _ in range(2)]
    pkg.gated_ff_grad(dh, x, w[:10], w[10:], out=kept, accumulate=True)
    assert all(bool((t == 1).all()) for t in kept)
    pkg.gated_ff_grad(dh, x, w[:10], w[10:], out=kept)
    assert not any(bool(t.any()) for t in kept)


@types
def test_far_activations(pkg, dev, dtype):
    """Gates far out on both sides: the activation is g or 0, its slope 1 or 0, and nothing is NaN."""
    far = 3e4 if dtype == torch.float16 else 1e6
    x = torch.tensor([[far], [-far], [100.0], [-100.0], [0.0]]).to(dtype)
    one = torch.ones(8, 1).to(dtype)
    for act in ACTS:
        h = pkg.gated_ff(x.to(dev), one.to(dev), (one / 512).to(dev), activation=act).double().cpu()
        want = torch.where(x > 0, x.double() * x.double() / 512, 0.0).expand(5, 8).clone()
        want[want > torch.finfo(dtype).max] = math.inf
        check(h, want, want.abs().nan_to_num(posinf=0) * 4 * UNIT[dtype] + 1e-30, act)
        got = pkg.gated_ff_grad(torch.ones(5, 8, device=dev).to(dtype), x.to(dev), one.to(dev), (one / 512).to(dev),
                                activation=act, weights=False)
        want = torch.where(x > 0, 8 * (x.double() / 512 + x.double() / 512), 0.0)
        check(got.dx, want, want.abs() * 8 * UNIT[dtype] + 1e-30, act)


@types
def test_unsound_rows_stay_alone(pkg, dev, dtype):
    """A row with a NaN or an infinity spoils its own results and the weights' gradients, no other row's."""
    n, width, inner = 300, 72, 100
    x, w, dh = operands(dtype, n, width, inner)
    x[7, 3], x[299, 71] = math.nan, math.inf
    x, w, dh = x.to(dev), w.to(dev), dh.to(dev)
    h = pkg.gated_ff(x, w[:inner], w[inner:])
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[7, 299]] = True
    assert not h[~bad.to(dev)].isnan().any() and h[7].isnan().all()
    clean = x.clone()
    clean[[7, 299]] = 0
    assert torch.equal(h[~bad.to(dev)], pkg.gated_ff(clean, w[:inner], w[inner:])[~bad.to(dev)])
    got = pkg.gated_ff_grad(dh, x, w[:inner], w[inner:])
    assert not got.dx[~bad.to(dev)].isnan().any() and got.dw_gate.isnan().any()


def test_differences(pkg, dev):
    """The gradients against difference quotients of the 64-bit forward formula."""
    x, w, dh = operands(torch.float32, 5, 6, 7)
    for act in ACTS:
        got = pkg.gated_ff_grad(dh.to(dev), x.to(dev), w[:7].to(dev), w[7:].to(dev), activation=act)
        step = 1e-5
        for name, t in zip(got._fields, (x, w[:7], w[7:])):
            for at in ((0, 0), (2, 3), (4, 5)):
                args = [v.double() for v in (x, w[:7], w[7:])]
                which = ("dx", "dw_gate", "dw_up").index(name)
                side = []
                for sign in (1, -1):
                    moved = [a.clone() for a in args]
                    moved[which][at] += sign * step
                    side.append(float((forward(*moved, act)[0] * dh.double()).sum()))
                slope = (side[0] - side[1]) / (2 * step)
                # a quotient's own error: step^2 times third derivatives of order 1, and 64-bit sums over 2 step
                assert abs(float(getattr(got, name)[at]) - slope) < 1e-5, (act, name, at)


def test_autograd(pkg, dev):
    x, w, dh = operands(torch.bfloat16, 33, 40, 56)
    leaf = [t.to(dev).requires_grad_() for t in (x, w[:56], w[56:])]
    h = pkg.gated_ff(*leaf, activation="gelu")
    h.backward(dh.to(dev))
    got = pkg.gated_ff_grad(dh.to(dev), *[t.detach() for t in leaf], activation="gelu")
    assert all(torch.equal(t.grad, g) for t, g in zip(leaf, got))
    alone = x.to(dev).requires_grad_()
    pkg.gated_ff(alone, leaf[1].detach(), leaf[2].detach(), activation="gelu").backward(dh.to(dev))
    assert torch.equal(alone.grad, leaf[0].grad)
    h = pkg.gated_ff(*leaf)
    with torch.no_grad():
        leaf[1].add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        h.sum().backward()
    with pytest.raises(ValueError, match="without gradients"):
        pkg.gated_ff(*leaf, out=torch.empty(33, 56, dtype=torch.bfloat16, device=dev))


def test_refusals(pkg, dev):
    x, w, dh = (t.to(dev) for t in operands(torch.bfloat16, 10, 16, 24))
    g, u = w[:24], w[24:]
    for call, what in (
            (lambda: pkg.gated_ff(x, g, u, activation="tanh"), "activation"),
            (lambda: pkg.gated_ff(x, g.float(), u), "w_gate must be"),
            (lambda: pkg.gated_ff(x, g, u[:5]), "24 rows, w_up 5"),
            (lambda: pkg.gated_ff(x, g[:, :8], u), "width 8"),
            (lambda: pkg.gated_ff(x, g.t(), u.t()), "width 24"),
            (lambda: pkg.gated_ff(x, g.t().contiguous().t(), u), "adjacent"),
            (lambda: pkg.gated_ff(x, g, u, out=torch.empty(10, 25, dtype=x.dtype, device=dev)), "shape"),
            (lambda: pkg.gated_ff(x, g, u, out=g[:10].new_empty(10, 24).float()), "must be"),
            (lambda: pkg.gated_ff(x[:, :0], g[:, :0], u[:, :0]), "positive"),
            (lambda: pkg.gated_ff(x.double(), g, u), "float32, bfloat16 or float16"),
            (lambda: pkg.gated_ff_grad(dh[:, :5], x, g, u), "dh has shape"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, dtype=torch.float16), "float32 or x's"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, inputs=False, weights=False), "neither"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, accumulate=True), "accumulate"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, out=[g.clone()]), "pair"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, out=[g, u]), "shares memory"),
            (lambda: pkg.gated_ff_grad(dh, x, g, u, out=[(t := g.clone()), t]), "shares memory"),
            (lambda: pkg.gated_ff(w.view(-1)[:160].view(10, 16), g, u, out=w.view(-1)[:240].view(10, 24)), "shares")):
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(pkg.ECError):
        pkg.gated_ff(torch.empty(1, (1 << 19) + 1, device=dev), torch.empty(1, (1 << 19) + 1, device=dev),
                     torch.empty(1, (1 << 19) + 1, device=dev))
