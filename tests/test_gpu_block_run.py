"""The block operators as they are used: a block and its update together against 64-bit autograd, on streams, in graphs,
past 2^32 elements, and on both sides of the rules that split products along their sums."""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT
from test_gpu_block_ff import forward, gradients, operands
from test_gpu_block_ortho import steps_of, tolerance, update
from test_gpu_step import E, UNIT, check, gen, rounded, types

pytestmark = pytest.mark.gpu


@types
@pytest.mark.parametrize("n,width,inner", [(100, 5000, 40), (70, 2100, 300), (3000, 40, 24), (40, 48, 3000), (2000, 129, 65),
                                           (260, 72, 2500)])
def test_split_sums(pkg, dev, dtype, n, width, inner):
    x, w, dh = operands(dtype, n, width, inner)
    want, bound, _ = forward(x, w[:inner], w[inner:], "silu")
    wd = w.to(dev)
    check(pkg.gated_ff(x.to(dev), wd[:inner], wd[inner:]), want, rounded(want, dtype, bound), "h")
    out = [torch.ones(inner, width, device=dev) for _ in range(2)]
    got = pkg.gated_ff_grad(dh.to(dev), x.to(dev), wd[:inner], wd[inner:], out=out, accumulate=True)
    wants = gradients(dh, x, w[:inner], w[inner:], "silu", dtype, torch.float32)
    check(got.dx, *wants[0], "dx")
    for g, (want, bound) in zip(got[1:], wants[1:]):
        check(g, want + 1.0, bound + 2 * E * (want.abs() + 1.0), "dw added to ones")


@types
@pytest.mark.parametrize("n,width,inner", [(777, 501, 1333), (30, 1000, 2665), (200, 330, 500), (50, 512, 2050), (1, 4100, 700),
                                           (520, 1030, 770)])
def test_sums_in_one_launch(pkg, dev, dtype, n, width, inner):
    """Both kinds of gradients in one launch, dx split or not, dW in middle or small tiles: as when they are asked for
    one at a time, within the same bounds, and nothing beside the rows written."""
    x, w, dh = operands(dtype, n, width, inner)
    xd, wd, dhd = x.to(dev), w.to(dev), dh.to(dev)
    for out in {dtype, torch.float32}:
        wants = gradients(dh, x, w[:inner], w[inner:], "silu", dtype, out)
        room = torch.full((2, inner, width + 9), 2.0, dtype=out, device=dev)
        into = [room[0, :, :width], room[1, :, :width]]
        both = pkg.gated_ff_grad(dhd, xd, wd[:inner], wd[inner:], out=into)
        alone = [pkg.gated_ff_grad(dhd, xd, wd[:inner], wd[inner:], weights=False).dx,
                 *pkg.gated_ff_grad(dhd, xd, wd[:inner], wd[inner:], inputs=False, dtype=out)[1:]]
        for got in (both, alone):
            for name, g, (want, bound) in zip(both._fields, got, wants):
                check(g, want, bound, name)
        assert bool((room[:, :, width:] == 2).all())
        again = pkg.gated_ff_grad(dhd, xd, wd[:inner], wd[inner:], dtype=out)
        assert all(torch.equal(a, b) for a, b in zip(both, again))


@pytest.mark.parametrize("shape", [(40, 6000), (6000, 40), (130, 3000), (2, 3000, 100)], ids=str)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_split_grams(pkg, dev, shape, out):
    x = update(torch.float32, *shape)
    want = steps_of(x.double())
    got = pkg.orthogonalize(x.to(dev), dtype=out).double().cpu()
    norm = want.norm(dim=(-2, -1))
    # (a bf16 result of 64 rows and more also has the products' roundings, below 2^-9 of it)
    assert bool(((got - want).norm(dim=(-2, -1)) <= tolerance(*shape[-2:], 5) + (1.01 * UNIT[out] + 2.0 ** -9) * norm).all())


def model(seed, vocab=64, width=96, inner=160, n=40, dtype=torch.bfloat16):
    g = gen("block", seed)
    r = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    return {"table": r(vocab, width).to(dtype), "first": (1 + 0.1 * r(width)).to(dtype),
            "w_gate": (r(inner, width) / math.sqrt(width)).to(dtype), "w_up": (r(inner, width) / math.sqrt(width)).to(dtype),
            "down": (r(inner, width) / math.sqrt(inner)).to(dtype), "post": (1 + 0.1 * r(width)).to(dtype),
            "gate": r(2, width).to(dtype), "last": (1 + 0.1 * r(width)).to(dtype),
            "head": (r(width, vocab) / math.sqrt(width)).to(dtype)}, torch.randint(0, vocab, (n,), generator=g), \
        torch.randint(0, vocab, (n,), generator=g)


def loss_of(ec, p, tokens, targets):
    """Embedding, norm, gated feed-forward, norms and gate around it, logits, log probabilities."""
    x = ec.embed(tokens, p["table"])
    r = ec.residual_norm(x, weight=p["first"])
    h = ec.gated_ff(r.normed, p["w_gate"], p["w_up"]) @ p["down"]
    r = ec.residual_norm(r.residual, h, gate=p["gate"], scale=0.5, branch_weight=p["post"], weight=p["last"])
    return ec.token_logprobs(r.normed @ p["head"], targets).logprobs.sum()


def exact_loss(p, tokens, targets, eps=1e-6):
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + eps).rsqrt()   # noqa: E731
    x = p["table"][tokens]
    z = rms(x) * p["first"]
    h = torch.nn.functional.silu(z @ p["w_gate"].T) * (z @ p["w_up"].T) @ p["down"]
    x = x + 0.5 * p["gate"].repeat_interleave(len(tokens) // 2, 0) * (rms(h) * p["post"])
    logits = rms(x) * p["last"] @ p["head"]
    return torch.log_softmax(logits, -1).gather(1, targets[:, None]).sum()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_block_in_a_step(pkg, dev, dtype):
    """Gradients of every parameter through the operators together, then their norm and the updates of the matrices."""
    p, tokens, targets = model(1, dtype=dtype)
    leaves = {k: v.to(dev).requires_grad_() for k, v in p.items()}
    got = loss_of(pkg, leaves, tokens.to(dev), targets.to(dev))
    got.backward()
    exact = {k: v.double().requires_grad_() for k, v in p.items()}
    want = exact_loss(exact, tokens, targets)
    want.backward()
    # eight roundings of the chain's tensors, each half a step, in the mean square of many values
    near = 8 * (UNIT[dtype] if dtype != torch.float32 else 64 * E)
    got, want = float(got.detach()), float(want.detach())
    assert abs(got - want) <= near * abs(want)
    for k, leaf in leaves.items():
        far = (leaf.grad.double().cpu() - exact[k].grad).norm() / exact[k].grad.norm()
        assert float(far) <= near, (k, float(far))
    grads = pkg.GradList([v.grad for v in leaves.values()])
    norm = grads.clip(1.0)
    assert bool(norm.isfinite())
    for k in ("w_gate", "w_up", "down"):
        leaf = leaves[k]
        before, version = leaf.detach().clone(), leaf._version
        with torch.no_grad():
            pkg.orthogonalize(leaf.grad, scale=-0.02, base=leaf, keep=0.998, out=leaf)
        assert leaf._version > version
        step = (leaf.detach().double() - 0.998 * before.double()).cpu() / -0.02
        want = steps_of(leaf.grad.double().cpu())
        # the weights' rounding, magnified, over all of them
        most = UNIT[dtype] * float(before.norm()) / 0.02 + tolerance(*leaf.shape, 5) + 2.0 ** -9 * float(want.norm())
        assert float((step - want).norm()) <= 1.5 * most, k


def everything(pkg, a):
    h = pkg.gated_ff(a["x"], a["wg"], a["wu"])
    g = pkg.gated_ff_grad(a["dh"], a["x"], a["wg"], a["wu"])
    r = pkg.residual_norm(a["x"], g.dx, gate=a["v"], branch_weight=a["v"], weight=a["v"])
    d = pkg.residual_norm_grad(a["x"], g.dx, r.residual, g.dx, rstd=r.rstd, branch_rstd=r.branch_rstd, gate=a["v"],
                               branch_weight=a["v"], weight=a["v"])
    return [h, *g, *r, *d, pkg.orthogonalize(g.dw_gate), pkg.orthogonalize(g.dw_up, dtype=torch.float32),
            pkg.gated_ff(a["x"][:7], a["wg"], a["wu"])]


def arguments(dev, n, width, inner, key=0):
    x, w, dh = (t.to(dev) for t in operands(torch.bfloat16, n, width, inner, key))
    return {"x": x, "wg": w[:inner], "wu": w[inner:], "dh": dh, "v": torch.ones_like(x[0])}


@pytest.mark.parametrize("n,width,inner", [(70, 65, 129), (300, 512, 96)])
def test_streams(pkg, dev, n, width, inner):
    a = arguments(dev, n, width, inner)
    want = everything(pkg, a)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = everything(pkg, a)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    h = pkg.gated_ff(a["x"], a["wg"], a["wu"], stream=side)
    g = pkg.gated_ff_grad(a["dh"], a["x"], a["wg"], a["wu"], stream=side)
    r = pkg.residual_norm(a["x"], a["x"], weight=a["v"], stream=side)
    o = pkg.orthogonalize(a["wg"], stream=side)
    side.synchronize()
    assert torch.equal(h, want[0]) and all(torch.equal(x, y) for x, y in zip(g, want[1:4]))
    assert torch.equal(o, pkg.orthogonalize(a["wg"]))
    assert torch.equal(r.normed, pkg.residual_norm(a["x"], a["x"], weight=a["v"]).normed)


def test_two_graphs(pkg, dev):
    """Two captured runs replayed in turns, with eager ones between."""
    runs = []
    for i, size in enumerate([(70, 65, 129), (300, 512, 96)]):
        a = arguments(dev, *size)
        everything(pkg, a)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = everything(pkg, a)
        runs.append((a, graph, out, size))
    for turn in range(1, 4):
        for a, graph, out, size in runs:
            for k, v in arguments(dev, *size, key=turn).items():
                a[k].copy_(v)
        torch.cuda.synchronize()
        for _, graph, _, _ in runs:
            graph.replay()
        torch.cuda.synchronize()
        for a, _, out, _ in runs:
            want = everything(pkg, a)
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_a_captured_backward(pkg, dev):
    """Forward and backward passes through autograd in one graph, replayed on new values between eager passes.  The leaves
    of the graph are its own: no eager graph of them lives while it is captured."""
    def pass_of(p):
        z = pkg.residual_norm(p["x"], weight=p["first"]).normed
        h = pkg.gated_ff(z, p["w_gate"], p["w_up"])
        r = pkg.residual_norm(p["x"][:, :32], h[:, :32].contiguous(), gate=p["gate"], branch_weight=p["post"], weight=p["last"])
        return torch.autograd.grad((r.residual, r.normed), list(p.values()), (p["x"].detach()[:, :32].contiguous(),) * 2)

    def values(key):
        g = gen("backward", key)
        shapes = {"x": (40, 72), "first": (72,), "w_gate": (48, 72), "w_up": (48, 72), "gate": (5, 32), "post": (32,), "last": (32,)}
        return {k: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev) for k, s in shapes.items()}

    side = torch.cuda.Stream(dev)
    leaves = {k: v.requires_grad_() for k, v in values(0).items()}
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        for _ in range(2):
            pass_of(leaves)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = pass_of(leaves)
    for key in range(1, 4):
        new = values(key)
        with torch.no_grad():
            for k, v in leaves.items():
                v.copy_(new[k])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = pass_of({k: v.requires_grad_() for k, v in new.items()})
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_past_32_bits(pkg, dev):
    """More than 2^32 elements of h, dh and the stream: the last rows are those of a call on them alone."""
    n, width, inner = 66000, 64, 65600
    x, w, _ = (t.to(dev) for t in operands(torch.bfloat16, n, width, inner))
    h = pkg.gated_ff(x, w[:inner], w[inner:])
    assert h.numel() > 1 << 32
    last = pkg.gated_ff(x[-300:], w[:inner], w[inner:])
    assert torch.equal(h[-300:], last)
    g = pkg.gated_ff_grad(h, x, w[:inner], w[inner:], weights=False)
    few = pkg.gated_ff_grad(last, x[-300:], w[:inner], w[inner:], weights=False)
    # other tiles add the sums in another order
    check(g.dx[-300:], few.dx, few.dx.double().abs().cpu() * 2 * UNIT[torch.bfloat16] + 1e-3 * float(few.dx.double().abs().max()), "dx")
    del g
    v = h.view(-1)[: h.numel() // 4096 * 4096].view(-1, 4096)
    r = pkg.residual_norm(v, v, weight=torch.ones(4096, dtype=v.dtype, device=dev), out=v)
    assert v.numel() > 1 << 32 and bool(r.rstd[-1].isfinite())
    tail = r.residual[-5:].clone()
    check((tail.double().square().mean(1) + 1e-6).rsqrt(), r.rstd[-5:].double(), 1e-2 * r.rstd[-5:].double().cpu(), "rstd")


def test_the_current_device_stays(pkg, dev):
    before = torch.cuda.current_device()
    everything(pkg, arguments(dev, 70, 65, 129))
    assert torch.cuda.current_device() == before


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_on_a_device_that_is_not_current(pkg, dev):
    want = everything(pkg, arguments(torch.device("cuda", 0), 70, 65, 129))
    with torch.cuda.device(0):
        got = everything(pkg, arguments(torch.device("cuda", 1), 70, 65, 129))
        assert torch.cuda.current_device() == 0
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


def test_gates_of_other_dimensions_are_refused(pkg, dev):
    x, v = torch.randn(6, 4, 8, device=dev), torch.ones(8, device=dev)
    same = pkg.residual_norm(x, x, gate=v, weight=v).normed
    for shape in ((1, 8), (1, 1, 8), (6, 8), (6, 1, 8), (6, 4, 8)):
        assert torch.equal(pkg.residual_norm(x, x, gate=torch.ones(shape, device=dev), weight=v).normed, same)
    for shape in ((4, 8), (1, 4, 8), (2, 8), (12, 8), (6, 2, 8), (1, 6, 4, 8)):
        with pytest.raises(ValueError, match="evenly"):
            pkg.residual_norm(x, x, gate=torch.ones(shape, device=dev), weight=v)


def test_train_block_example(pkg, dev):
    path = os.path.join(ROOT, "megatron-lm_amd", "examples", "train_block.py")
    spec = importlib.util.spec_from_file_location("train_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert math.isfinite(mod.main(steps=4))
