"""The norms around a block and their gradients on the GPU against 64-bit formulas: widths from one element to the longest,
odd and strided rows, every type, gates for all rows, for groups and for each row.

Bounds.  e = 2^-24.  A sum of n terms in fp32 is off by at most n e of its sum of magnitudes; a row's factor
1 / rms, from such a sum, a division and a reciprocal root, by (width / 2 + 4) e relative."""
import math

import pytest
import torch

from test_gpu_step import E, check, gen, rounded, types

pytestmark = pytest.mark.gpu

EPS = 1e-6


def operands(dtype, n, width, gates, post, pre, key=0):
    g = gen("norms", n, width, gates, post, pre, key)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    return {"residual": (3 * r(n, width)).to(dtype), "branch": r(n, width).to(dtype),
            "gate": r(gates, width).to(dtype) if gates else None,
            "branch_weight": (1 + 0.3 * r(width)).to(dtype) if post else None,
            "weight": (1 + 0.3 * r(width)).to(dtype) if pre else None}


def spread(gate, n):
    return 1.0 if gate is None else gate.double().repeat_interleave(n // gate.shape[0], 0)


def forward(o, scale):
    r, y = o["residual"].double(), o["branch"].double()
    n, width = r.shape
    root = (width / 2 + 4) * E
    brstd = (y.square().mean(1) + EPS).rsqrt()
    u = y * brstd[:, None] * o["branch_weight"].double() if o["branch_weight"] is not None else y
    added = scale * spread(o["gate"], n) * u
    total = r + added
    off = added.abs() * (root + 6 * E) + 2 * E * total.abs()
    rstd = (total.square().mean(1) + EPS).rsqrt()
    # the sum's error moves its root mean square by at most its own
    far = root + off.square().mean(1).sqrt() * rstd
    result = {"residual": (total, off), "branch_rstd": (brstd, brstd * root), "rstd": (rstd, rstd * far * 1.01)}
    if o["weight"] is not None:
        w = o["weight"].double()
        normed = total * rstd[:, None] * w
        result["normed"] = normed, (off * rstd[:, None] * w.abs() + normed.abs() * (far[:, None] + 4 * E)) * 1.01
    return result


def gradients(o, total, ds, dn, rstd, brstd, scale):
    """{name: (value, bound of its fp32 value)}; total, rstd and brstd as the call gets them."""
    d = ds.double() if ds is not None else torch.zeros_like(total, dtype=torch.float64)
    y = o["branch"].double()
    n, width = y.shape
    off = torch.zeros_like(d)
    out = {}

    def norm_back(t, hat, root, extra):
        """root * (t - hat mean(t hat)) and its bound, where t is off by `extra`."""
        s = (t * hat).mean(1, keepdim=True)
        es = ((width + 6) * E * (t * hat).abs() + extra * hat.abs()).mean(1, keepdim=True)
        value = root * (t - hat * s)
        return value, root * (extra + hat.abs() * es + 6 * E * (t.abs() + (hat * s).abs()))

    if dn is not None:
        w = o["weight"].double()
        hat = total.double() * rstd.double()[:, None]
        t = dn.double() * w
        value, bound = norm_back(t, hat, rstd.double()[:, None], 2 * E * t.abs())
        d, off = d + value, bound + 2 * E * (d.abs() + value.abs())
        terms = dn.double() * hat
        out["weight"] = terms.sum(0), (n + 4) * E * terms.abs().sum(0)
    out["residual"] = d, off
    post = o["branch_weight"] is not None
    root = brstd.double()[:, None] if post else 1.0
    hat = y * root
    bw = o["branch_weight"].double() if post else 1.0
    gate = spread(o["gate"], n)
    if o["gate"] is not None:
        terms, bound = scale * d * hat * bw, abs(scale) * off * (hat * bw).abs()
        rows = o["gate"].shape[0]
        total_of = lambda t: t.reshape(rows, n // rows, width).sum(1)   # noqa: E731
        out["gate"] = total_of(terms), total_of(bound + (n // rows + 8) * E * (terms.abs() + bound))
    g = scale * gate * d
    eg = torch.as_tensor(abs(scale) * gate).abs() * off + 4 * E * g.abs()
    if post:
        terms, bound = g * hat, eg * hat.abs()
        out["branch_weight"] = terms.sum(0), (bound + (n + 8) * E * (terms.abs() + bound)).sum(0)
        value, bound = norm_back(g * bw, hat, root, eg * bw.abs() + 2 * E * (g * bw).abs())
        out["branch"] = value, bound
    else:
        out["branch"] = g, eg
    return out


WIDTHS = [1, 2, 7, 8, 33, 64, 255, 512, 513, 1024, 1999, 2048, 2500, 4096, 5001, 8192]
FORMS = [(0, True, True), (1, False, True), (1, True, True), (-1, True, True), (3, True, True), (3, True, False), (0, False, False)]


@types
@pytest.mark.parametrize("width", WIDTHS)
def test_both_directions(pkg, dev, dtype, width):
    for at, (gates, post, pre) in enumerate(FORMS):
        n = (6, 21, 3)[(at + width) % 3]
        gates = n if gates < 0 else gates
        o = operands(dtype, n, width, gates, post, pre)
        scale = 0.37
        on = {k: None if v is None else v.to(dev) for k, v in o.items()}
        r = pkg.residual_norm(on["residual"], on["branch"], gate=on["gate"], scale=scale, eps=EPS,
                              branch_weight=on["branch_weight"], weight=on["weight"])
        want = forward(o, scale)
        assert (r.normed is not None) == (r.rstd is not None) == pre and (r.branch_rstd is not None) == post
        for name, got in zip(r._fields, r):
            if got is not None:
                value, bound = want[name]
                check(got, value, rounded(value, got.dtype, bound), (name, width, n, gates, post))
        g = gen("dnorms", n, width)
        ds, dn = (torch.randn(n, width, generator=g).to(dtype) for _ in range(2))
        for a, b in ((ds, dn), (ds, None), (None, dn)):
            b = b if pre else None
            if a is None and b is None:
                continue
            got = pkg.residual_norm_grad(None if a is None else a.to(dev), None if b is None else b.to(dev), r.residual,
                                         on["branch"], rstd=r.rstd, branch_rstd=r.branch_rstd, gate=on["gate"], scale=scale,
                                         branch_weight=on["branch_weight"], weight=on["weight"])
            wants = gradients(o, r.residual.cpu(), a, b, None if r.rstd is None else r.rstd.cpu(),
                              None if r.branch_rstd is None else r.branch_rstd.cpu(), scale)
            for name, v in zip(got._fields, got):
                assert (v is not None) == (name in wants), name
                if v is not None:
                    value, bound = wants[name]
                    check(v, value, rounded(value, v.dtype, bound * 1.05), (name, width, n, gates, post))


@pytest.mark.parametrize("n,width,gates", [(5000, 64, 1), (4099, 40, 0), (3000, 520, 3000), (2400, 100, 600), (2400, 100, 800),
                                           (1200, 2048, 4), (1, 16384, 1), (2, 12000, 2), (1040, 8200, 1)])
def test_many_rows_and_long_ones(pkg, dev, n, width, gates):
    """Column sums over teams of every kind: parts of a gate's rows, whole gates, more gates than teams."""
    dtype = torch.bfloat16 if n % 2 == 0 else torch.float32
    o = operands(dtype, n, width, gates, True, True)
    on = {k: None if v is None else v.to(dev) for k, v in o.items()}
    r = pkg.residual_norm(on["residual"], on["branch"], gate=on["gate"], branch_weight=on["branch_weight"], weight=on["weight"])
    for name, (value, bound) in forward(o, 1.0).items():
        got = getattr(r, name)
        check(got, value, rounded(value, got.dtype, bound), name)
    g = gen("dnorms", n, width)
    ds, dn = (torch.randn(n, width, generator=g).to(dtype) for _ in range(2))
    got = pkg.residual_norm_grad(ds.to(dev), dn.to(dev), r.residual, on["branch"], rstd=r.rstd, branch_rstd=r.branch_rstd,
                                 gate=on["gate"], branch_weight=on["branch_weight"], weight=on["weight"])
    for name, (value, bound) in gradients(o, r.residual.cpu(), ds, dn, r.rstd.cpu(), r.branch_rstd.cpu(), 1.0).items():
        v = getattr(got, name)
        check(v, value, rounded(value, v.dtype, bound * 1.05), name)
    again = pkg.residual_norm_grad(ds.to(dev), dn.to(dev), r.residual, on["branch"], rstd=r.rstd, branch_rstd=r.branch_rstd,
                                   gate=on["gate"], branch_weight=on["branch_weight"], weight=on["weight"])
    assert all(torch.equal(a, b) for a, b in zip(got, again) if a is not None)


@types
def test_norm_alone(pkg, dev, dtype):
    """A first block's norm: no branch."""
    o = operands(dtype, 9, 300, 0, False, True)
    o["branch"] = torch.zeros_like(o["residual"])
    x = o["residual"].to(dev)
    r = pkg.residual_norm(x, weight=o["weight"].to(dev), eps=EPS)
    assert r.residual is x and r.branch_rstd is None
    want = forward(o, 1.0)
    for name in ("normed", "rstd"):
        check(getattr(r, name), want[name][0], rounded(want[name][0], getattr(r, name).dtype, want[name][1]), name)
    dn = torch.randn(9, 300, generator=gen("alone")).to(dtype)
    got = pkg.residual_norm_grad(None, dn.to(dev), x, rstd=r.rstd, weight=o["weight"].to(dev))
    assert got.branch is None and got.gate is None and got.branch_weight is None
    wants = gradients(o, o["residual"], None, dn, r.rstd.cpu(), None, 1.0)
    for name in ("residual", "weight"):
        check(getattr(got, name), wants[name][0], rounded(wants[name][0], getattr(got, name).dtype, wants[name][1] * 1.05), name)


@types
def test_strides_and_place(pkg, dev, dtype):
    o = operands(dtype, 12, 130, 3, True, True)
    on = {k: v.to(dev) for k, v in o.items()}
    rest = dict(gate=on["gate"].view(3, 1, 130), branch_weight=on["branch_weight"], weight=on["weight"])
    want = pkg.residual_norm(on["residual"], on["branch"], **rest)
    wide = torch.full((12, 400), 2.0, dtype=dtype, device=dev)
    a, b, c = wide[:, 1:131], wide[:, 140:270], wide[:, 270:400]
    a.copy_(on["residual"]), b.copy_(on["branch"])
    got = pkg.residual_norm(a, b, out=c, **rest)
    assert torch.equal(got.residual, want.residual) and torch.equal(got.normed, want.normed)
    assert bool((wide[:, 0] == 2).all()) and bool((wide[:, 131:140] == 2).all())
    version = wide._version
    assert torch.equal(pkg.residual_norm(a, b, out=a, **rest).residual, want.residual) and wide._version > version
    assert torch.equal(a, want.residual)
    grads = pkg.residual_norm_grad(on["residual"], on["branch"], want.residual, on["branch"], rstd=want.rstd,
                                   branch_rstd=want.branch_rstd, **rest)
    d1, d2, d3 = (torch.empty(12, 133, dtype=dtype, device=dev)[:, 3:] for _ in range(3))
    d1.copy_(on["residual"]), d2.copy_(on["branch"]), d3.copy_(want.residual)
    again = pkg.residual_norm_grad(d1, d2, d3, b, rstd=want.rstd, branch_rstd=want.branch_rstd, **rest)
    assert grads.gate.shape == (3, 1, 130) and all(torch.equal(x, y) for x, y in zip(grads, again))


def test_no_rows(pkg, dev):
    w = torch.ones(16, device=dev)
    x = torch.empty(0, 16, device=dev)
    r = pkg.residual_norm(x, x.clone(), gate=w, branch_weight=w, weight=w)
    assert r.residual.shape == r.normed.shape == (0, 16) and r.rstd.shape == (0,)
    g = pkg.residual_norm_grad(x, x, x, x.clone(), rstd=r.rstd, branch_rstd=r.branch_rstd, gate=w, branch_weight=w, weight=w)
    assert g.residual.shape == (0, 16) and not any(bool(t.any()) for t in (g.gate, g.branch_weight, g.weight))


@types
def test_zero_rows_and_unsound_ones(pkg, dev, dtype):
    """A row of zeros has a finite factor and no NaN; a row with a NaN or infinity spoils its own values only."""
    o = operands(dtype, 10, 100, 0, True, True)
    o["residual"][2], o["branch"][2] = 0, 0
    o["residual"][5, 7], o["branch"][8, 99] = math.nan, math.inf
    on = {k: None if v is None else v.to(dev) for k, v in o.items()}
    r = pkg.residual_norm(on["residual"], on["branch"], branch_weight=on["branch_weight"], weight=on["weight"])
    assert not r.residual[2].any() and not r.normed[2].any()
    check(r.rstd[2], torch.tensor(1 / math.sqrt(EPS)), 1e3 * 8 * E)
    good = [i for i in range(10) if i not in (5, 8)]
    assert r.normed[5].isnan().all() and r.normed[8].isnan().any() and bool(r.normed[good].isfinite().all())
    ones = torch.ones_like(on["residual"])
    g = pkg.residual_norm_grad(ones, ones, r.residual, on["branch"], rstd=r.rstd, branch_rstd=r.branch_rstd,
                               branch_weight=on["branch_weight"], weight=on["weight"])
    assert bool(g.residual[good].isfinite().all()) and bool(g.branch[[0, 1, 3, 4, 6, 7, 9]].isfinite().all())
    assert g.weight.isnan().any()


@pytest.mark.parametrize("post", [False, True])
def test_autograd_and_differences(pkg, dev, post):
    """Through autograd, the gradients against difference quotients of the 64-bit forward formula."""
    n, width, scale = 6, 10, 0.8
    o = operands(torch.float32, n, width, 2, post, True)
    ca, cb = (torch.randn(n, width, generator=gen(k)) for k in "ab")
    leaves = {k: v.to(dev).requires_grad_() for k, v in o.items() if v is not None}
    r = pkg.residual_norm(leaves["residual"].view(2, 3, width), leaves["branch"].view(2, 3, width),
                          gate=leaves["gate"].view(2, 1, width), scale=scale, branch_weight=leaves.get("branch_weight"),
                          weight=leaves["weight"])
    assert r.residual.shape == (2, 3, width) and not r.rstd.requires_grad
    ((r.residual.view(n, width) * ca.to(dev)).sum() + (r.normed.view(n, width) * cb.to(dev)).sum()).backward()

    def loss(o):
        f = forward(o, scale)
        return float((f["residual"][0] * ca).sum() + (f["normed"][0] * cb).sum())

    for name, leaf in leaves.items():
        for at in ((0, 0), (1, 7)):
            at = at[1:] if leaf.dim() == 1 else at
            side = []
            for sign in (1, -1):
                moved = {k: None if v is None else v.double().clone() for k, v in o.items()}
                moved[name][at] += sign * 1e-6
                side.append(loss(moved))
            # the quotient's own error: 64-bit sums of order 100 over 2e-6, and fp32's in the gradient
            assert abs(float(leaf.grad[at]) - (side[0] - side[1]) / 2e-6) < 5e-5, (name, at)
    only = o["residual"].to(dev).requires_grad_()
    r = pkg.residual_norm(only, weight=leaves["weight"])
    assert r.residual is only
    r.normed.sum().backward()
    want = pkg.residual_norm_grad(None, torch.ones(n, width, device=dev), only.detach(), rstd=r.rstd, weight=leaves["weight"].detach())
    assert torch.equal(only.grad, want.residual)


def test_refusals(pkg, dev):
    x, y, w = torch.randn(6, 20, device=dev), torch.randn(6, 20, device=dev), torch.ones(20, device=dev)
    for call, what in (
            (lambda: pkg.residual_norm(x), "neither"), (lambda: pkg.residual_norm(x, gate=w, weight=w), "go with a branch"),
            (lambda: pkg.residual_norm(x, y.half(), weight=w), "branch must be"),
            (lambda: pkg.residual_norm(x, y[:3], weight=w), "shape"), (lambda: pkg.residual_norm(x, y, weight=w[:5]), "shape"),
            (lambda: pkg.residual_norm(x, y, gate=torch.ones(4, 20, device=dev)), "evenly"),
            (lambda: pkg.residual_norm(x, y, gate=torch.ones(20, 1, device=dev)), "gate must be"),
            (lambda: pkg.residual_norm(x, y, scale=math.inf), "finite"), (lambda: pkg.residual_norm(x, y, eps=-1.0), "eps"),
            (lambda: pkg.residual_norm(x, y, out=torch.empty(6, 21, device=dev)), "shape"),
            (lambda: pkg.residual_norm(x[:3], y[:3], out=x.view(-1)[10:70].view(3, 20)), "shares"),
            (lambda: pkg.residual_norm(x, y, gate=x[:1], out=x), "shares memory with gate"),
            (lambda: pkg.residual_norm(x.t(), y.t(), weight=w[:6]), "adjacent"),
            (lambda: pkg.residual_norm_grad(None, None, x), "neither"),
            (lambda: pkg.residual_norm_grad(None, x, x), "weight and rstd"),
            (lambda: pkg.residual_norm_grad(x, None, x, y, branch_weight=w), "branch_rstd"),
            (lambda: pkg.residual_norm_grad(x, None, x, gate=w), "go with a branch"),
            (lambda: pkg.residual_norm_grad(x[:2], None, x, y), "shape"),
            (lambda: pkg.residual_norm_grad(x, x, x, y, weight=w, rstd=w[:6].half()), "rstd must be")):
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(ValueError, match="without gradients"):
        pkg.residual_norm(x.clone().requires_grad_(), y, weight=w, out=torch.empty_like(x))
    with pytest.raises(pkg.ECError):
        pkg.residual_norm(torch.empty(1, 16385, device=dev), weight=torch.ones(16385, device=dev))
