"""A language model of a few blocks trained with the framework's operators alone between its library products: embedding,
norms around gated feed-forward blocks, the loss, clipping, and orthogonalised updates of the blocks' matrices.

    python megatron-lm_amd/examples/train_block.py [steps]

Each block normalises the stream (``residual_norm``), takes the gated feed-forward of it (``gated_ff``, gate and up weights
in one buffer), and adds it back through a norm and a learned gate; ``residual_norm`` does that and the next block's norm in one
pass.  The gradients are clipped into an fp32 buffer (``GradList.clip``); the blocks' matrices take the orthogonalised momentum
(``orthogonalize``, onto their decayed fp32 master weights, in place), the other parameters a step along the sign of
theirs.  A step whose norm is not finite is skipped.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import __graft_entry__  # noqa: E402

VOCAB, HIDDEN, INNER, BLOCKS, BATCH, SEQ = 512, 128, 256, 2, 16, 64
LR, MOMENTUM, DECAY, MAX_NORM = 0.02, 0.9, 0.01, 1.0


def parameters(gen, dev):
    """Names and fp32 master weights; a block's matrices are those of two dimensions."""
    def normal(*shape):
        return torch.empty(shape, device=dev).normal_(0.0, shape[-1] ** -0.5, generator=gen)
    p = {"table": normal(VOCAB, HIDDEN), "out": normal(HIDDEN, VOCAB), "norm.last": torch.ones(HIDDEN, device=dev)}
    for b in range(BLOCKS):
        p[f"block{b}.up"] = normal(2 * INNER, HIDDEN)
        p[f"block{b}.down"] = normal(INNER, HIDDEN)
        p[f"norm{b}.before"] = torch.ones(HIDDEN, device=dev)
        p[f"norm{b}.after"] = torch.ones(HIDDEN, device=dev)
        p[f"norm{b}.gate"] = torch.ones(HIDDEN, device=dev)
    return p


def logits_of(ec, w, tokens):
    r = ec.residual_norm(ec.embed(tokens, w["table"], scale=HIDDEN ** 0.5), weight=w["norm0.before"])
    for b in range(BLOCKS):
        up = w[f"block{b}.up"]
        h = ec.gated_ff(r.normed, up[:INNER], up[INNER:]) @ w[f"block{b}.down"]
        following = w[f"norm{b + 1}.before"] if b + 1 < BLOCKS else w["norm.last"]
        r = ec.residual_norm(r.residual, h, gate=w[f"norm{b}.gate"], scale=(2 * BLOCKS) ** -0.5,
                             branch_weight=w[f"norm{b}.after"], weight=following)
    return r.normed @ w["out"]


def main(steps: int = 60) -> float:
    ec = __graft_entry__.load_package()
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(0)
    master = parameters(gen, dev)
    weights = {k: v.bfloat16().requires_grad_() for k, v in master.items()}
    momenta = {k: torch.zeros_like(v) for k, v in master.items()}
    for w in weights.values():
        w.grad = torch.zeros_like(w)
    grads = {k: torch.zeros_like(v) for k, v in master.items()}
    grad_list = ec.GradList([w.grad for w in weights.values()], out=list(grads.values()))
    loss = None
    for step in range(1, steps + 1):
        start = torch.randint(0, VOCAB, (BATCH, 1), device=dev, generator=gen)
        tokens = (start + 7 * torch.arange(SEQ + 1, device=dev)) % VOCAB
        for w in weights.values():
            w.grad.zero_()
        logits = logits_of(ec, weights, tokens[:, :-1].contiguous())
        mean = -ec.token_logprobs(logits, tokens[:, 1:].contiguous()).logprobs.mean()
        mean.backward()
        norm = grad_list.clip(MAX_NORM)
        if not bool(norm.isfinite()):
            print(f"step {step}: gradient norm {float(norm)}, skipped", flush=True)
            continue
        for k, m in master.items():
            momenta[k].lerp_(grads[k], 1 - MOMENTUM)
            if k.startswith("block"):
                ec.orthogonalize(momenta[k], scale=-LR * max(1.0, m.shape[0] / m.shape[1]) ** 0.5, base=m,
                                 keep=1 - LR * DECAY, out=m)
            else:
                m.sub_(0.1 * LR * momenta[k].sign())
            weights[k].data.copy_(m)
        loss = float(mean.detach())
        if step == 1 or step % 20 == 0:
            print(f"step {step}: loss {loss:.3f}, gradient norm {float(norm):.3f}", flush=True)
    print(f"train_block ok: loss {loss:.3f} after {steps} steps", flush=True)
    return loss


if __name__ == "__main__":
    main(*[int(a) for a in sys.argv[1:2]])
