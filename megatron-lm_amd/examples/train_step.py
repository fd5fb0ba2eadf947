"""A training loop around the engine's saves: the step's operators, a snapshot, a loss of slices and
the load, on one GPU.

    python megatron-lm_amd/examples/train_step.py [steps]

A small language model (embedding, one gated layer, output weights) learns to repeat a cyclic
sequence.  Each step looks the tokens up (``embed``), takes the loss over the vocabulary
(``token_logprobs``, with its entropy logged), lets autograd bring the gradients back through both,
clips them to a norm of a quarter (``GradList.clip``, from bf16 into the fp32 buffer that Adam
reads) and skips the update where the norm is not finite.  Then the state (bf16 weights, fp32 master weights and
moments) is coded as RS(4,2) slices by ``GpuSliceCodec.snapshot``, two slices are lost, and the state
rebuilt from the others has to give a probe batch the same log probabilities, bit for bit.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import __graft_entry__  # noqa: E402

VOCAB, HIDDEN, BATCH, SEQ = 512, 128, 16, 64
LR, BETAS, EPS, MAX_NORM = 1e-3, (0.9, 0.95), 1e-8, 0.25


def logits_of(ec, weights, tokens):
    table, gate, up, out = weights
    x = ec.embed(tokens, table, scale=HIDDEN ** 0.5)
    x = x + torch.nn.functional.silu(x @ gate) * (x @ up)
    return x @ out


def probe(ec, weights, tokens):
    """Log probabilities, entropies and likeliest tokens of a batch's next tokens."""
    with torch.no_grad():
        return ec.token_logprobs(logits_of(ec, weights, tokens[:, :-1].contiguous()),
                                 tokens[:, 1:].contiguous(), entropy=True, top=3)


def main(steps: int = 60) -> float:
    ec = __graft_entry__.load_package()
    from megatron_lm_amd.checkpoint import GpuSliceCodec
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(0)

    shapes = [(VOCAB, HIDDEN), (HIDDEN, HIDDEN), (HIDDEN, HIDDEN), (HIDDEN, VOCAB)]
    sizes = [a * b for a, b in shapes]
    master = [torch.empty(s, device=dev).normal_(0.0, 0.05, generator=gen) for s in shapes]
    weights = [m.bfloat16().requires_grad_() for m in master]
    moment, square = ([torch.zeros_like(m) for m in master] for _ in range(2))
    # the gradients stay where they are from step to step, so their list is made once
    for w in weights:
        w.grad = torch.zeros_like(w)
    grads = torch.zeros(sum(sizes), device=dev)
    main_grads = [g.view(s) for g, s in zip(grads.split(sizes), shapes)]
    grad_list = ec.GradList([w.grad for w in weights], out=main_grads)

    def batch():
        start = torch.randint(0, VOCAB, (BATCH, 1), device=dev, generator=gen)
        return (start + 7 * torch.arange(SEQ + 1, device=dev)) % VOCAB

    first = loss = None
    for step in range(1, steps + 1):
        tokens = batch()
        for w in weights:
            w.grad.zero_()
        r = ec.token_logprobs(logits_of(ec, weights, tokens[:, :-1].contiguous()),
                              tokens[:, 1:].contiguous(), entropy=True)
        mean = -r.logprobs.mean()
        mean.backward()
        norm = grad_list.clip(MAX_NORM)
        if not bool(norm.isfinite()):   # an unsound step: no update, and no snapshot of it
            print(f"step {step}: gradient norm {float(norm)}, skipped", flush=True)
            continue
        for m, w, g, a, b in zip(master, weights, main_grads, moment, square):
            a.lerp_(g, 1 - BETAS[0])
            b.lerp_(g * g, 1 - BETAS[1])
            m.sub_(LR * (a / (1 - BETAS[0] ** step)) / ((b / (1 - BETAS[1] ** step)).sqrt() + EPS))
            w.data.copy_(m)
        loss = float(mean.detach())
        first = loss if first is None else first
        if step == 1 or step % 20 == 0:
            print(f"step {step}: loss {loss:.3f}, entropy {float(r.entropy.detach().mean()):.3f}, gradient norm "
                  f"{float(norm):.3f}", flush=True)

    state = [w.detach() for w in weights] + master + moment + square
    codec = GpuSliceCodec(4, 2, 4096)
    meta, slices = codec.snapshot(state).result(timeout=60)
    asked = batch()
    before = probe(ec, weights, asked)
    lost = (1, 4)
    loaded = codec.decode(meta, {p: s for p, s in enumerate(slices) if p not in lost}, dev)
    after = probe(ec, loaded[:len(weights)], asked)
    for name, a, b in zip(before._fields, before, after):
        if not torch.equal(a, b):
            raise AssertionError(f"{name} differs after the load")
    print(f"train_step ok: loss {first:.3f} -> {loss:.3f} in {steps} steps; slices {lost} lost, the loaded state "
          f"answers as the saved one", flush=True)
    return loss


if __name__ == "__main__":
    main(*[int(a) for a in sys.argv[1:2]])
