"""Operators of a block of the model between the embedding and the loss, and of its matrices' update.

``gated_ff`` and ``gated_ff_grad`` (the gated feed-forward: both projections, the activation and the
product), ``residual_norm`` and ``residual_norm_grad`` (a block's branch normalised, gated, scaled and added to
the residual stream, and the sum normalised for the next block), and ``orthogonalize`` (an update
orthogonalised by Newton-Schulz products, scaled and added to the decayed weights).  With ``embed``,
``token_logprobs`` and ``GradList`` they make a training step of the matrices that the engine protects.

Every function takes HIP tensors of float32, bfloat16 or float16, sums in fp32 (products on the matrix
cores), rounds once where it stores unless it says otherwise, and enqueues on the given stream or torch's current one, through
the C ABI of ``include/ec_mi355.h``.  The same inputs give the same bits.  With gradients enabled,
``gated_ff`` and ``residual_norm`` are differentiable functions of all their tensors, backward only: a forward-mode
tangent is refused.  The other three have no gradient, and refuse tensors that require one but under
``torch.no_grad()``.  A backward pass is captured into a HIP graph, as with torch's own operators, while no eager
pass's results of the same leaves are held.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .step import _TYPES, _call, _finite

_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _activation(name: str) -> int:
    if name not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {name!r}")
    return _ACTIVATIONS[name]


def _differentiable(*tensors) -> bool:
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def _plain(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.detach()


# ------------------------------------------------------ gated feed-forward --

class GatedGrads(NamedTuple):
    """What ``gated_ff_grad`` returns; None where it was not asked for."""
    dx: Optional[torch.Tensor]
    dw_gate: Optional[torch.Tensor]
    dw_up: Optional[torch.Tensor]


class _GatedFf(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.activation = activation
        return gated_ff(x.detach(), w_gate.detach(), w_up.detach(), activation=activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up = (t.detach() for t in ctx.saved_tensors)
        need = ctx.needs_input_grad
        weights = need[1] or need[2]
        g = gated_ff_grad(dh.contiguous(), x, w_gate, w_up, activation=ctx.activation, inputs=need[0],
                          weights=weights)
        return g.dx, g.dw_gate if need[1] else None, g.dw_up if need[2] else None, None


def gated_ff(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *, activation: str = "silu",
             out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """act(x @ w_gate.T) * (x @ w_up.T), of shape [*x.shape[:-1], inner], in one kernel.

    ``x`` is [..., width] (contiguous, or two-dimensional with strided rows); the weights are [inner,
    width], rows may be strided, so they can be the halves of one buffer.  ``activation`` is "silu"
    (g * sigmoid(g)), "gelu" (g * Phi(g)) or "gelu_tanh" (its tanh form)."""
    code = _activation(activation)
    if _differentiable(x, w_gate, w_up):
        if out is not None or stream is not None:
            raise ValueError("out and stream are for calls without gradients")
        return _GatedFf.apply(x, w_gate, w_up, activation)
    return _call("ec_gated_ff", _lib.shards().gated_ff, x, stream, x, w_gate, w_up, code, out)[0]


def gated_ff_grad(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *,
                  activation: str = "silu", inputs: bool = True, weights: bool = True,
                  dtype: Optional[torch.dtype] = None, out: Optional[Sequence[torch.Tensor]] = None,
                  accumulate: bool = False, stream=None) -> GatedGrads:
    """The gradients of ``gated_ff`` from that of its result, ``dh``: with respect to x (``inputs``) and both
    weights (``weights``).  The projections are computed again, so nothing but x and the weights is kept
    from the forward pass.

    The weights' gradients are of ``dtype``, x's type (the default) or float32, or of that of ``out``, a pair
    of tensors that they are written to, or with ``accumulate`` added to (a micro-batch's part of a gradient buffer).
    The gradients of the two projections, which the products read, are rounded to x's type (in fp16, past 65504, to
    infinities, and results are not finite); with 256 rows or fewer, whose roundings average out less, their rounding errors
    are taken along."""
    if not inputs and not weights:
        raise ValueError("neither the inputs' nor the weights' gradients are asked for")
    if dtype is not None and dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    if out is not None and len(out) != 2:
        raise ValueError("out must be a pair of tensors")
    pair = (None, None) if out is None else tuple(out)
    for t in pair:
        if dtype is not None and getattr(t, "dtype", dtype) != dtype:
            raise ValueError(f"out is {t.dtype}, dtype {dtype}")
    dtype = dtype or getattr(x, "dtype", None)
    return GatedGrads(*_call(
        "ec_gated_ff_grad", _lib.shards().gated_ff_grad, x, stream, dh, x, w_gate, w_up, _activation(activation),
        bool(inputs), bool(weights), _TYPES.get(dtype, 0), *pair, accumulate)[:3])


# ------------------------------------------------- norms around a block --

class ResidualNorm(NamedTuple):
    """What ``residual_norm`` returns."""
    residual: torch.Tensor                 # the stream with the branch added
    normed: Optional[torch.Tensor]         # the next block's input
    rstd: Optional[torch.Tensor]           # one over the root mean square of the stream's rows, fp32; no gradient
    branch_rstd: Optional[torch.Tensor]    # that of the branch's rows


class ResidualNormGrads(NamedTuple):
    """What ``residual_norm_grad`` returns: the gradients of the stream and the branch in their type, those of the gate
    and the weights in fp32; None where there is no such input."""
    residual: torch.Tensor
    branch: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    branch_weight: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, gate, branch_weight, weight, scale, eps):
        r = residual_norm(residual.detach(), _plain(branch), gate=_plain(gate), scale=scale,
                          branch_weight=_plain(branch_weight), weight=_plain(weight), eps=eps)
        total = residual if branch is None else r.residual
        ctx.save_for_backward(total, branch, gate, branch_weight, weight, r.rstd, r.branch_rstd)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (r.rstd, r.branch_rstd) if t is not None])
        return (None if branch is None else r.residual, *r[1:])

    @staticmethod
    @once_differentiable
    def backward(ctx, dresidual, dnormed, _rstd, _branch_rstd):
        if dresidual is None and dnormed is None:
            return (None,) * 7
        total, branch, gate, branch_weight, weight, rstd, branch_rstd = map(_plain, ctx.saved_tensors)
        g = residual_norm_grad(None if dresidual is None else dresidual.contiguous(),
                               None if dnormed is None else dnormed.contiguous(), total, branch, rstd=rstd,
                               branch_rstd=branch_rstd, gate=gate, scale=ctx.scale, branch_weight=branch_weight,
                               weight=weight)
        cast = lambda d, t: d if d is None else d.to(t.dtype)   # noqa: E731
        return (g.residual, g.branch, cast(g.gate, gate), cast(g.branch_weight, branch_weight),
                cast(g.weight, weight), None, None)


def residual_norm(residual: torch.Tensor, branch: Optional[torch.Tensor] = None, *,
                  gate: Optional[torch.Tensor] = None, scale: float = 1.0,
                  branch_weight: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                  eps: float = 1e-6, out: Optional[torch.Tensor] = None, stream=None) -> ResidualNorm:
    """What stands between two blocks, in one pass:

        u = branch, or branch_weight * branch / rms(branch) with ``branch_weight`` (a norm after the block)
        residual' = residual + scale * gate * u
        normed = weight * residual' / rms(residual')    with ``weight`` (the norm before the next block)

    with rms(v) = sqrt(mean(v^2) + eps) over the last dimension, at most 16384 wide.  ``residual`` and ``branch``
    are [..., width] of one type (contiguous, or two-dimensional with strided rows), the weights [width].  ``gate`` has rows
    that theirs share evenly, in order: one for all ([width]), one for each sequence of [batch, length, width] ([batch,
    width] or [batch, 1, width]: the leading dimensions are the gate's), or one for each row; with two-dimensional rows
    any number that divides theirs.  Without a
    ``branch`` only the norm is taken (a first block's).  normed is that of the sum before its rounding.
    ``out`` takes the sum, and may be the residual itself."""
    scale, eps = _finite(scale, "scale"), _finite(eps, "eps")
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if _differentiable(residual, branch, gate, branch_weight, weight):
        if out is not None or stream is not None:
            raise ValueError("out and stream are for calls without gradients")
        r = ResidualNorm(*_ResidualNorm.apply(residual, branch, gate, branch_weight, weight, scale, eps))
    else:
        r = ResidualNorm(*_call("ec_residual_norm", _lib.shards().residual_norm, residual, stream, residual, branch,
                                gate, scale, branch_weight, weight, eps, out))
    return r if branch is not None else r._replace(residual=residual)


def residual_norm_grad(dresidual: Optional[torch.Tensor], dnormed: Optional[torch.Tensor], total: torch.Tensor,
                       branch: Optional[torch.Tensor] = None, *, rstd: Optional[torch.Tensor] = None,
                       branch_rstd: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                       scale: float = 1.0, branch_weight: Optional[torch.Tensor] = None,
                       weight: Optional[torch.Tensor] = None, stream=None) -> ResidualNormGrads:
    """The gradients of ``residual_norm`` from those of its stream (``dresidual``) and its normed rows (``dnormed``;
    one of them may be None), with the stream ``total``, ``rstd`` and ``branch_rstd`` that it returned and the
    branch, gate and weights that it was given.  The weights' and the gate's are sums over rows in fixed places."""
    return ResidualNormGrads(*_call(
        "ec_residual_norm_grad", _lib.shards().residual_norm_grad, total, stream, dresidual, dnormed, total, branch,
        rstd, branch_rstd, gate, _finite(scale, "scale"), branch_weight, weight)[:5])


# ------------------------------------------------- orthogonalised updates --

def orthogonalize(x: torch.Tensor, *, steps: int = 5, coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, scale: float = 1.0, base: Optional[torch.Tensor] = None, keep: float = 1.0,
                  dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """keep * base + scale * X for each matrix of ``x`` ([..., rows, cols], contiguous, or one with strided rows), where X
    is x / (|x| + eps) after ``steps`` Newton-Schulz steps

        X <- a X + (b A + c A A) X,   A = X X.T   (from the right, with X.T X, for tall matrices)

    with a, b, c the ``coefficients``: the singular values s go through a s + b s^3 + c s^5, those of the default
    towards 1.  |x| is the root of the sum of squares.  Without ``base`` the result is scale * X.

    A weight update in place: ``orthogonalize(momentum, scale=-lr, base=weight, keep=1 - lr * decay, out=weight)``.
    The result is of ``out``'s type, or ``dtype``, or the base's, or x's; base and out are of the same.  Products
    are of values of 22 bits with fp32 sums; for a bf16 result with 64 or more rows and columns of
    11 bits, added to a X with 22, which leaves about 1e-3 of the result, up to 3e-3 where x has a single nonzero row
    (``dtype=torch.float32`` takes 22 whatever x is).  The coefficients are of magnitude up to 1024, and may
    take singular values from 1 to 2^-30 or 2^20 before the last step (results of larger ones may be infinite or NaN, of
    smaller ones zeros).  A value that is not finite makes its matrix NaN."""
    steps = int(steps)
    if not 1 <= steps <= 64:
        raise ValueError(f"steps must be between 1 and 64, got {steps}")
    a, b, c = (_finite(v, "coefficients") for v in coefficients)
    if max(abs(a), abs(b), abs(c)) > 1024:
        raise ValueError("coefficients must not exceed 1024 in magnitude")
    if _finite(eps, "eps") <= 0:
        raise ValueError(f"eps must be positive, got {eps}")
    if dtype is not None and dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    if out is not None and dtype is not None and getattr(out, "dtype", dtype) != dtype:
        raise ValueError(f"out is {out.dtype}, dtype {dtype}")
    return _call("ec_orthogonalize", _lib.shards().orthogonalize, x, stream, x, steps, a, b, c, eps,
                 _finite(scale, "scale"), base, _finite(keep, "keep"), -1 if dtype is None else _TYPES[dtype], out)[0]
