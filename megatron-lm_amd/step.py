"""Operators of the training step around the saves.

What a training loop computes between two saves on the tensors that the engine
protects: ``embed`` and ``embed_grad`` (rows of the embedding table by token, and
the table's gradient), ``token_logprobs`` and ``token_logprobs_grad`` (the loss over
the vocabulary: log probabilities of given tokens, entropy, the likeliest tokens),
and ``grad_norm`` / ``clip_grads`` / ``GradList`` (the global norm of a gradient list
and its clipping).  The norm says whether a step is sound: where it is not finite a loop
skips the update, and the snapshot after it; and the log probabilities of a
probe batch say whether a loaded state answers as the saved one did.

Every function takes HIP tensors of float32, bfloat16 or float16, computes in
fp32 (sums of squares in fp64), rounds once where it stores, and enqueues on the
given stream or torch's current one, through the C ABI of
``include/ec_mi355.h``.  The same inputs give the same bits.  With gradients enabled,
``embed`` and ``token_logprobs`` are differentiable functions of the table and
the logits.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .codec import _raw_stream
from .layout import _hold, _upload

MAX_TOP = 16   # alternatives token_logprobs returns at most

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _finite(v: float, what: str) -> float:
    v = float(v)
    if not math.isfinite(v):
        raise ValueError(f"{what} must be finite, got {v}")
    return v


def _call(name: str, fn, tensor, stream, *args):
    """The binding's ``fn(*args)`` on ``stream`` or torch's current one: what it returned after the
    status.  Memory for a caller's own stream comes from that stream's share of the caching
    allocator (a block of the current stream's may still be in use there), and is not handed
    out again before work enqueued on the current stream, which reads the results, is done."""
    if stream is None:
        status, *made = fn(*args)
    else:
        device = getattr(tensor, "device", None)
        _raw_stream(stream, device)   # the devices agree
        current = torch.cuda.current_stream(device)
        with torch.cuda.stream(stream):
            status, *made = fn(*args)
        _hold(current, *[t for t in made if t is not None])
    if status != _lib.EC_OK:
        _lib.check(status, name)
    return made


# --------------------------------------------------------------- embedding --

class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, vocab_start):
        ctx.save_for_backward(tokens)
        ctx.like = table.shape[0], table.dtype, scale, vocab_start
        return embed(tokens, table.detach(), scale=scale, vocab_start=vocab_start)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (tokens,) = ctx.saved_tensors
        vocab, dtype, scale, start = ctx.like
        return embed_grad(tokens, dout.contiguous(), vocab, scale=scale, vocab_start=start,
                          dtype=dtype), None, None, None


def embed(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, vocab_start: int = 0,
          out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """scale * table[tokens - vocab_start], of shape [*tokens.shape, hidden] and the table's type.

    ``table`` is a rank's slice [vocabulary, hidden] of the embedding (rows may be
    strided); a token outside it gives a row of zeros, so the ranks' results
    add up to the whole lookup.  ``tokens`` are contiguous int32 or int64 of any
    shape."""
    if torch.is_grad_enabled() and isinstance(table, torch.Tensor) and table.requires_grad:
        if out is not None or stream is not None:
            raise ValueError("out and stream are for calls without gradients")
        return _Embed.apply(table, tokens, scale, vocab_start)
    return _call("ec_embed", _lib.shards().embed, table, stream,
                 tokens, table, _finite(scale, "scale"), vocab_start, out)[0]


def embed_grad(tokens: torch.Tensor, dout: torch.Tensor, vocab_size: int, *, scale: float = 1.0,
               vocab_start: int = 0, dtype: Optional[torch.dtype] = None,
               out: Optional[torch.Tensor] = None, accumulate: bool = False,
               stream=None) -> torch.Tensor:
    """The gradient [vocab_size, hidden] of ``embed``'s table: for each row scale times the sum of
    ``dout`` ([*tokens.shape, hidden]) over the positions of its token.

    ``dtype`` is float32 (the default) or dout's, or that of ``out``.  The tokens are
    sorted and each row's positions added in fp32, without atomics: in ascending order within tiles
    of 16 or 32 sorted positions, then a long run's tiles in a fixed grouping.
    ``accumulate`` adds to ``out`` and leaves the rows of tokens that do not occur untouched
    (a micro-batch's part of a gradient buffer); otherwise they are zeros."""
    dtype = torch.float32 if dtype is None else dtype
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    return _call("ec_embed_grad", _lib.shards().embed_grad, dout, stream,
                 tokens, dout, vocab_size, _finite(scale, "scale"), vocab_start, _TYPES[dtype], out,
                 accumulate)[0]


# ------------------------------------------------------- log probabilities --

class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, fp32 (and int64 tokens), in the shape of the targets."""
    logprobs: torch.Tensor                 # of the targets; 0 where there is none
    lse: torch.Tensor                      # log of the sum of exp(scale * logits); no gradient
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]   # [..., top], descending; no gradient
    top_tokens: Optional[torch.Tensor]     # [..., top], equal ones by ascending index


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, scale, entropy, top):
        r = token_logprobs(logits.detach(), targets, scale=scale, entropy=entropy, top=top)
        ctx.save_for_backward(logits, targets, r.lse, r.entropy)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (r.lse, r.top_logprobs, r.top_tokens) if t is not None])
        return tuple(r)

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogprobs, _lse, dentropy, _top, _tokens):
        logits, targets, lse, entropy = ctx.saved_tensors
        if dlogprobs is None and dentropy is None:
            return None, None, None, None, None
        dlogprobs = torch.zeros_like(lse) if dlogprobs is None else dlogprobs.contiguous()
        with_entropy = dentropy is not None
        d = token_logprobs_grad(logits.detach(), targets, lse, dlogprobs, scale=ctx.scale,
                                entropy=entropy if with_entropy else None,
                                dentropy=dentropy.contiguous() if with_entropy else None)
        return d, None, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, scale: float = 1.0,
                   entropy: bool = False, top: int = 0, stream=None) -> TokenLogprobs:
    """Log probabilities of ``targets`` (int64, the logits' leading shape) under the softmax of
    scale * ``logits`` ([..., vocabulary], contiguous, or two-dimensional with strided rows), in one
    pass over the logits, and on request the entropy and the ``top`` (at most MAX_TOP) likeliest tokens.

    With gradients enabled the log probabilities and the entropy are differentiable; ``lse`` and the
    alternatives are constants, so a term of the loss made from them (a penalty on lse) has
    no gradient.  The logits are those of the whole vocabulary: of a rank's slice the values are the
    slice's own, and a target in another slice would count as ignored, with no gradient for this one.

    A target outside the vocabulary (an ignored position) has log probability 0.  Logits
    of -infinity are masked; a row of nothing else has log probability and lse -infinity and
    entropy 0.  A NaN or +infinity makes its row's values NaN.  ``scale`` (one over the
    temperature) is positive."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        if stream is not None:
            raise ValueError("stream is for calls without gradients")
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, scale, entropy, top))
    return TokenLogprobs(*_call("ec_token_logprobs", _lib.shards().token_logprobs, logits, stream,
                                logits, targets, _positive(scale, "scale"), bool(entropy), top))


def _positive(v: float, what: str) -> float:
    if _finite(v, what) <= 0:
        raise ValueError(f"{what} must be positive, got {v}")
    return float(v)


def token_logprobs_grad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor,
                        dlogprobs: torch.Tensor, *, entropy: Optional[torch.Tensor] = None,
                        dentropy: Optional[torch.Tensor] = None, scale: float = 1.0,
                        out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The gradient with respect to the logits, from the gradients of ``token_logprobs``' log
    probabilities and (``dentropy``, together with the ``entropy`` it returned) entropies, in the
    logits' type.  Probabilities are exp(scale * logits - ``lse``), at most 1.  ``out`` may be the logits themselves.  Ignored positions have no part in
    ``dlogprobs``; masked logits, and rows of nothing else, have gradient 0."""
    return _call("ec_token_logprobs_grad", _lib.shards().token_logprobs_grad, logits, stream,
                 logits, targets, lse, dlogprobs, entropy, dentropy, _positive(scale, "scale"),
                 out)[0]


# ---------------------------------------------------------- gradient lists --

def _norm_code(norm_type) -> int:
    if norm_type == 2:
        return 2
    if norm_type in (math.inf, "inf"):
        return 0
    raise ValueError(f"norm_type must be 2 or infinity, got {norm_type!r}")


class GradList:
    """A list of gradient tensors (contiguous, on one device, any mix of types and sizes) prepared
    once for ``norm`` and ``clip``: a training loop keeps its gradient buffers, and the list of
    their pieces stays on the device.  ``clip`` writes to the tensors of ``out`` (same element
    counts, any of the types: bf16 gradients into fp32 ones), or in place; no two of the tensors
    written may overlap.  The list keeps the tensors alive; gradients that are replaced by other tensors need a new
    list.  Making one costs 0.3 to 2 us a tensor on the host (and an upload), more than the calls on small ones."""

    _clips = True

    def __init__(self, grads: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None):
        self.grads = list(grads)
        self.out = None if out is None else list(out)
        items, self._written = _lib.shards().grad_items(self.grads, self.out, self._clips)
        self.device = self.grads[0].device if self.grads else \
            torch.device("cuda", torch.cuda.current_device())
        with torch.cuda.device(self.device):
            self._items = _upload(items.numpy(), self.device)
            self.uploaded = torch.cuda.Event()
            self.uploaded.record()
        self._made_on = _raw_stream(None, self.device)

    def _run(self, what, stream, *args) -> torch.Tensor:
        if _raw_stream(stream, self.device) != self._made_on:
            on = torch.cuda.current_stream(self.device) if stream is None else stream
            on.wait_event(self.uploaded)
            _hold(on, self._items)
        return _call(what, _lib.shards().grad_call, self._items, stream, self._items, self._written,
                     *args)[0]

    def norm(self, norm_type: float = 2.0, *, grad_scale: float = 1.0, stream=None) -> torch.Tensor:
        """The norm of grad_scale times all elements, a 0-d fp32 tensor: the square root of the sum
        of squares, or (``norm_type`` infinity) the largest magnitude.  Not finite if an element
        is not."""
        return self._run("ec_grad_norm", stream, _finite(grad_scale, "grad_scale"),
                         _norm_code(norm_type), None, None)

    def clip(self, max_norm: float, norm_type: float = 2.0, *, grad_scale: float = 1.0,
             norm: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """Scales the gradients by grad_scale * min(1, max_norm / (norm + 1e-6)) and returns the
        norm (before clipping, of the scaled gradients).  ``norm`` (fp32, one value on the device) is used instead
        of this list's own: the norm over all ranks, reduced from each rank's ``norm()``.  Where the
        norm is not finite the gradients are scaled by grad_scale only."""
        if not float(max_norm) > 0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        return self._run("ec_grad_clip", stream, _finite(grad_scale, "grad_scale"),
                         _norm_code(norm_type), float(max_norm), norm)


class _NormList(GradList):
    """A list that is only read: its tensors may overlap."""
    _clips = False


def grad_norm(grads: Sequence[torch.Tensor], norm_type: float = 2.0, *, grad_scale: float = 1.0,
              stream=None) -> torch.Tensor:
    """``GradList(grads).norm(...)``, for a list that is used once.  Nothing is written, so the tensors
    may overlap, and one that is in the list twice counts twice."""
    return _NormList(grads).norm(norm_type, grad_scale=grad_scale, stream=stream)


def clip_grads(grads: Sequence[torch.Tensor], max_norm: float, norm_type: float = 2.0, *,
               grad_scale: float = 1.0, norm: Optional[torch.Tensor] = None,
               out: Optional[Sequence[torch.Tensor]] = None, stream=None) -> torch.Tensor:
    """``GradList(grads, out).clip(...)``, for a list that is used once."""
    return GradList(grads, out).clip(max_norm, norm_type, grad_scale=grad_scale, norm=norm,
                                     stream=stream)
