"""Norms of lists whose tensors overlap: a norm writes nothing."""
import math

import pytest
import torch

from test_gpu_step import E, gen

pytestmark = pytest.mark.gpu


def test_norm_of_tensors_that_overlap(pkg, dev):
    buf = torch.randn(40_000, generator=gen("overlap")).to(dev)
    lists = [[buf, buf], [buf[:30_000], buf[10_000:]], [buf[5:6], buf[:20_000], buf[5:6]], [buf, buf.view(200, 200)]]
    for grads in lists:
        flat = torch.cat([t.reshape(-1) for t in grads]).double()
        want = float(flat.norm())
        assert abs(float(pkg.grad_norm(grads)) - want) <= 2 * E * want
        assert float(pkg.grad_norm(grads, math.inf)) == float(flat.abs().max())
        # what a clip would write twice stays refused
        for call in (lambda: pkg.clip_grads(grads, 1.0), lambda: pkg.GradList(grads)):
            with pytest.raises(ValueError, match="shares memory"):
                call()
