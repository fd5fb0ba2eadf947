"""The block operators' edges on the host, without a GPU: every call returns before any device work, so the addresses are
never touched."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("kind", [0, 1, 2], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("width,inner", [(2048, 8192), (256, 256), (64, 512), (448, 64), (65, 4001), (1, 1)])
def test_gated_ff_without_rows(pkg, kind, width, inner):
    """No rows at widths whose sums are split along k with rows: no workspace, and nothing to do but the weights' zeros."""
    L = pkg._lib.lib()
    rows = (P, width, P, width, P, width, kind, 0, width, inner)
    assert L.ec_gated_ff_workspace(*rows, 0) == L.ec_gated_ff_workspace(*rows, 1) == 0
    assert L.ec_gated_ff(*rows, 0, P, inner, None, 0, None) == pkg._lib.EC_OK
    assert L.ec_gated_ff_grad(P, inner, *rows, 0, P, width, P, width, P, width, kind, 1, None, 0, None) == pkg._lib.EC_OK
    assert L.ec_gated_ff_grad(P, inner, *rows, 0, P, width, None, 0, None, 0, kind, 0, None, 0, None) == pkg._lib.EC_OK


@pytest.mark.parametrize("accumulate", [0, 1])
def test_the_input_gradient_of_no_rows(pkg, accumulate):
    """A dx without elements has no address: nothing asked for is refused where there are rows only."""
    L = pkg._lib.lib()

    def call(n):
        return L.ec_gated_ff_grad(P, 48, P, 32, P, 32, P, 32, 1, n, 32, 48, 0, None, 32, None, 0, None, 0, 1, accumulate, P,
                                  1 << 20, None)

    assert call(0) == pkg._lib.EC_OK and call(4) == pkg._lib.EC_EINVAL


def test_tangents_are_refused(pkg):
    """Forward-mode derivatives are not had, and not dropped either: of every operand, of the step's operators too."""
    w, v, p = torch.ones(4, 8), torch.ones(8), torch.ones(3, 4)
    tokens = torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(3, 8), torch.ones(3, 8))
        for call in (lambda: pkg.gated_ff(x, w, w), lambda: pkg.gated_ff_grad(p, x, w, w),
                     lambda: pkg.residual_norm(x, weight=v), lambda: pkg.residual_norm_grad(x, None, x, x),
                     lambda: pkg.orthogonalize(x), lambda: pkg.embed(tokens, x), lambda: pkg.token_logprobs(x, tokens)):
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
            with pytest.raises(ValueError, match="tangent"):
                call()


def test_calls_without_gradients_of_their_own_refuse_operands_that_need_one(pkg):
    """With gradients enabled their results would be cut from the graph; not under no_grad, where an update belongs."""
    x, p, w, v, r = torch.ones(3, 8), torch.ones(3, 4), torch.ones(4, 8), torch.ones(8), torch.ones(3)
    calls = {
        "gated_ff_grad": (lambda **k: pkg.gated_ff_grad(*k.values()), dict(dh=p, x=x, w_gate=w, w_up=w)),
        "residual_norm_grad": (lambda dr, dn, t, b, **k: pkg.residual_norm_grad(dr, dn, t, b, **k),
                               dict(dr=x, dn=x, t=x, b=x, rstd=r, branch_rstd=r, gate=v, branch_weight=v, weight=v)),
        "orthogonalize": (lambda x, **k: pkg.orthogonalize(x, **k), dict(x=w, base=w, out=w))}
    for name, (call, operands) in calls.items():
        for which in operands:
            one = {k: t.clone().requires_grad_() if k == which else t for k, t in operands.items()}
            with pytest.raises(ValueError, match=f"{name} has no gradient"):
                call(**one)
            with torch.no_grad(), pytest.raises(ValueError, match="device"):   # host tensors, and nothing else
                call(**one)
        with pytest.raises(ValueError, match="device"):
            call(**operands)
    with pytest.raises(ValueError, match="gated_ff_grad has no gradient"):
        pkg.gated_ff_grad(p, x, w, w, out=(w, w.clone().requires_grad_()))


def test_a_dtype_other_than_that_of_out_is_refused(pkg):
    x, p, w = (torch.ones(s, dtype=torch.bfloat16) for s in ((3, 8), (3, 4), (4, 8)))
    for out in ((w, w), (w.float(), w), (w, w.float())):
        with pytest.raises(ValueError, match="out is torch.bfloat16, dtype torch.float32"):
            pkg.gated_ff_grad(p, x, w, w, dtype=torch.float32, out=out)
    for dtype in (None, torch.bfloat16):   # the host tensors are what is left to refuse
        with pytest.raises(ValueError, match="device"):
            pkg.gated_ff_grad(p, x, w, w, dtype=dtype, out=(w, w))


def test_a_pair_in_one_tensor_is_a_pair(pkg):
    x, p, w = torch.ones(3, 8), torch.ones(3, 4), torch.ones(4, 8)
    with pytest.raises(ValueError, match="device"):
        pkg.gated_ff_grad(p, x, w, w, out=torch.ones(2, 4, 8))
    with pytest.raises(ValueError, match="pair"):
        pkg.gated_ff_grad(p, x, w, w, out=torch.ones(0, 4, 8))
