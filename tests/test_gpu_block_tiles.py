"""The block operators' products in every tile and split that calls of many rows and large matrices take, with ends inside a
tile in every direction, against 64-bit products.  Beside each size stand the tiles and splits that the host
chooses for it; a host test asks the rule itself for them, so that no change of its costs moves a size away unseen."""
import pytest
import torch

from test_gpu_block_ff import forward, gradients, operands
from test_gpu_block_ortho import fast_steps_of, steps_of, update
from test_gpu_step import E, UNIT, check, rounded

pytestmark = pytest.mark.gpu

# type ("narrow": bf16 and fp16), rows, width, inner; shape / splits of the projections, of dx and of both dW
FF = [("narrow", 1503, 200, 4100, "large/1 least/2 middle/1"), ("narrow", 303, 521, 4100, "middle/1 least/4 large/1"),
      ("narrow", 4100, 520, 4100, "large/1 middle/3 large/2"), ("narrow", 4100, 2100, 301, "middle/1 large/1 middle/2"),
      ("narrow", 2101, 2100, 1333, "least/1 large/3 middle/1"), ("narrow", 4101, 521, 299, "middle/1 middle/1 least/2"),
      ("narrow", 2100, 203, 2100, "middle/1 least/3 middle/3"),
      ("narrow", 257, 8300, 4100, "large/3 large/3 large/1"), ("narrow", 65, 4201, 4100, "middle/3 middle/6 middle/1"),
      ("narrow", 130, 8301, 131, "least/9 least/1 large/1"),
      ("fp32", 1503, 201, 4100, "large/1 least/4 least/1"), ("fp32", 777, 1100, 1333, "middle/3 least/1 least/1"),
      ("fp32", 1500, 203, 2100, "middle/1 least/4 middle/3"), ("fp32", 300, 2100, 777, "least/3 least/3 middle/1"),
      ("fp32", 1501, 2100, 300, "least/4 middle/1 least/1"), ("fp32", 4100, 200, 777, "middle/1 middle/3 least/4"),
      ("fp32", 8150, 2041, 500, "middle/1 large/1 least/1"), ("fp32", 300, 2041, 4090, "least/2 least/3 large/1"),
      ("fp32", 1100, 4201, 2100, "large/3 least/1 middle/1"), ("fp32", 65, 8300, 2100, "least/6 middle/6 middle/1")]

# kind (fast: bf16 results; exact: the others), batch, rows, cols; of A, B and X
ORTHO = [("fast", 12, 2100, 1100, "large/1 large/1 large/1"), ("fast", 12, 1100, 2100, "large/1 large/1 large/1"),
         ("fast", 2, 2100, 3001, "large/2 middle/1 large/1"), ("fast", 2, 3001, 2100, "large/2 middle/1 large/1"),
         ("fast", 12, 1100, 1100, "large/1 large/1 middle/1"), ("fast", 12, 300, 1100, "least/1 least/1 large/1"),
         ("fast", 12, 1100, 301, "least/1 least/1 large/1"), ("fast", 12, 777, 520, "middle/1 middle/1 middle/1"),
         ("fast", 12, 523, 781, "middle/1 middle/1 middle/1"), ("fast", 3, 777, 2100, "middle/3 least/1 middle/1"),
         ("fast", 3, 2101, 777, "middle/3 least/1 middle/1"), ("fast", 3, 301, 1101, "least/1 least/1 middle/1"),
         ("fast", 1, 301, 523, "least/1 least/1 least/1"),
         ("exact", 12, 777, 520, "middle/1 middle/1 middle/1"), ("exact", 12, 523, 781, "middle/1 middle/1 middle/1"),
         ("exact", 3, 777, 2100, "middle/3 least/1 middle/1"), ("exact", 3, 2101, 777, "middle/3 least/1 middle/1"),
         ("exact", 8, 781, 300, "least/1 least/1 middle/1"), ("exact", 3, 257, 262, "least/1 least/1 least/1")]

TYPES = {"narrow": [torch.bfloat16, torch.float16], "fp32": [torch.float32]}


@pytest.mark.parametrize("dtype,n,width,inner", [(t, *c[1:4]) for c in FF for t in TYPES[c[0]]], ids=str)
def test_gated_ff(pkg, dev, dtype, n, width, inner):
    """Forward; dx and dW written beside other values, and dW added to ones in fp32."""
    x, w, dh = (t.to(dev) for t in operands(dtype, n, width, inner))
    gate, up = w[:inner], w[inner:]
    want, bound, _ = forward(x, gate, up, "silu")
    check(pkg.gated_ff(x, gate, up), want, rounded(want, dtype, bound).cpu(), "h")
    room = torch.full((2, inner, width + 9), 2.0, dtype=dtype, device=dev)
    got = pkg.gated_ff_grad(dh, x, gate, up, out=[room[0, :, :width], room[1, :, :width]])
    for name, g, (value, most) in zip(got._fields, got, gradients(dh, x, gate, up, "silu", dtype, dtype)):
        check(g, value, most.cpu(), name)
    assert bool((room[:, :, width:] == 2).all())
    ones = [torch.ones(inner, width, device=dev) for _ in range(2)]
    got = pkg.gated_ff_grad(dh, x, gate, up, out=ones, accumulate=True)
    wants = gradients(dh, x, gate, up, "silu", dtype, torch.float32)
    check(got.dx, wants[0][0], wants[0][1].cpu(), "dx")
    for g, (value, most) in zip(ones, wants[1:]):
        check(g, value + 1.0, (most + 2 * E * (value.abs() + 1.0)).cpu(), "dw added to ones")


@pytest.mark.parametrize("kind,batch,rows,cols", [c[:4] for c in ORTHO], ids=str)
def test_orthogonalize(pkg, dev, kind, batch, rows, cols):
    """As a whole and by rows and columns, so that an end that is lost in the norm of all is seen.

    A fast result is within twice the error of the same roundings made in 64 bits, a row's or column's, sums of hundreds of
    independent roundings, within three times the largest one's; beside its own rounding.  An exact one is within eight times
    the error of the same steps in fp32, whose values have 24 bits where pairs have 22."""
    x = update(torch.bfloat16 if batch % 2 else torch.float32, batch, rows, cols).to(dev)
    out = torch.bfloat16 if kind == "fast" else torch.float32
    base = torch.randn(batch, rows, cols, device=dev).to(out)
    got = pkg.orthogonalize(x, dtype=out)
    added = base.clone()
    assert pkg.orthogonalize(x, scale=-0.5, base=added, keep=0.75, out=added) is added
    for i in range(batch):
        want = steps_of(x[i].double())
        if kind == "fast":
            near, times = fast_steps_of(x[i].double()) - want, (2, 3)
        else:
            near, times = steps_of(x[i].cpu().float()).to(dev).double() - want, (8, 8)
        for result, value, scale in ((got[i], want, 1.0), (added[i], 0.75 * base[i].double() - 0.5 * want, 0.5)):
            far, own = result.double() - value, 1.01 * UNIT[out] * value.abs() + 2 * E * value.abs()
            assert bool(far.isfinite().all())
            assert float(far.norm()) <= times[0] * scale * float(near.norm()) + float(own.norm()), i
            for d in (0, 1):
                most = times[1] * scale * near.norm(dim=d).max() + own.norm(dim=d)
                assert bool((far.norm(dim=d) <= most).all()), (i, d, float((far.norm(dim=d) - most).max()))
