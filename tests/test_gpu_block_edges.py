"""The block operators' edges on the GPU: empty batches."""
import pytest
import torch

from test_gpu_step import types

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
