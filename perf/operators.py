"""The operators of a training step around the engine's saves, one pass each: their plain forms in elementary torch
operations, and the calls a user makes of the framework.

  embed     rows of an embedding table by token, scaled; tokens outside the rank's slice of the vocabulary give zeros
  egrad     the table's gradient: for each token the scaled sum of its positions' output gradients
  logp      log probabilities of given tokens, the log of the sum, the entropy, the likeliest tokens
  lgrad     the gradient of log probabilities and entropies with respect to the logits
  clip      the global 2-norm of a list of gradients, and the list scaled to at most a given norm
  norm      the norm alone

Tokens follow a Zipf distribution (the r-th commonest with probability ~ 1 / (r + 2.7)), with the ranks spread over the
vocabulary's ids, as text's do.  Logits are normal with the given token's raised.  Gradients are normal values whose
spread differs from tensor to tensor.
"""
import math
import random

import numpy as np
import torch

own = False

VOCAB, HIDDEN, LAYERS, SEQ = 50304, 2048, 24, 2048   # the 1.3B-parameter GPT of the engine's benchmark
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORED = -100
EPS = 1e-6


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


def listed():
    return [
        # one decoding step of a probe of eight sequences after a load: latency only
        {"name": "embed_8", "op": "embed", "n": 8, "vocab": VOCAB, "hidden": HIDDEN, "type": "bf16",
         "ids": "int64", "slices": 1},
        # a training step's micro-batch: 16 sequences of 2048 tokens
        {"name": "embed_32k", "op": "embed", "n": 16 * SEQ, "vocab": VOCAB, "hidden": HIDDEN, "type": "bf16",
         "ids": "int64", "slices": 1},
        # one sequence, an odd width, a rank that holds an eighth of the vocabulary: most tokens are others'
        {"name": "egrad_2k_slice", "op": "egrad", "n": SEQ, "vocab": VOCAB // 8, "hidden": 1999, "type": "fp32",
         "out": "fp32", "ids": "int32", "slices": 8},
        # the whole table's fp32 gradient from a step's 65536 tokens, the commonest on a tenth of the positions
        {"name": "egrad_64k", "op": "egrad", "n": 32 * SEQ, "vocab": VOCAB, "hidden": HIDDEN, "type": "bf16",
         "out": "fp32", "ids": "int64", "slices": 1},
        # sampling's log probabilities: a few rows, the likeliest five
        {"name": "logp_16_top5", "op": "logp", "n": 16, "vocab": VOCAB, "live": VOCAB, "type": "bf16",
         "top": 5, "entropy": False},
        # a step's loss over four sequences, with the entropy that training logs
        {"name": "logp_8k", "op": "logp", "n": 4 * SEQ, "vocab": VOCAB, "live": VOCAB, "type": "bf16",
         "top": 0, "entropy": True},
        # an odd vocabulary padded with masked columns, fp32 logits at a temperature, and eight alternatives
        {"name": "logp_700_top8", "op": "logp", "n": 700, "vocab": 32063, "live": 32001, "type": "fp32",
         "top": 8, "entropy": True},
        # the gradient of the small odd one, entropy bonus included
        {"name": "lgrad_513", "op": "lgrad", "n": 513, "vocab": 32063, "live": 32001, "type": "fp32",
         "entropy": True},
        # the gradient of a step's loss
        {"name": "lgrad_8k", "op": "lgrad", "n": 4 * SEQ, "vocab": VOCAB, "live": VOCAB, "type": "bf16",
         "entropy": False},
        # adapters and norms: many small gradients in bf16, clipped into fp32
        {"name": "clip_small", "op": "clip", "list": "ragged", "n": 120, "lo": 16, "hi": 32768, "type": "bf16",
         "out": "fp32", "sizes": 1},
        # the norm of a ragged mid-size list (its sizes are any, so tensors start at any element)
        {"name": "norm_ragged", "op": "norm", "list": "ragged", "n": 700, "lo": 1000, "hi": 4_000_000, "type": "bf16",
         "out": "bf16", "sizes": 2},
        # the whole model's fp32 gradients
        {"name": "clip_1300m", "op": "clip", "list": "gpt", "n": LAYERS, "lo": 0, "hi": 0, "type": "fp32",
         "out": "fp32", "sizes": 3},
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _width(rng, lo, hi):
    """A size between lo and hi, odd in half of the cases, else 32 past a multiple of 64 or a power of two."""
    n = _log(rng, lo, hi)
    how = rng.random()
    if how < 0.5:
        return n | 1
    return max(lo, n // 64 * 64 + 32) if how < 0.75 else 1 << max(4, n.bit_length() - 1)


def draw(rng):
    op = rng.choice(["embed", "egrad", "egrad", "logp", "logp", "lgrad", "clip", "norm"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("embed", "egrad"):
        hidden = _width(rng, 16, 8192)
        vocab = _log(rng, 300, min(160_000, 200_000_000 // hidden))
        n = _log(rng, 1, min(131_072, 130_000_000 // hidden))
        case = {"op": op, "n": n, "vocab": vocab, "hidden": hidden, "type": kind,
                "ids": rng.choice(["int32", "int64"]), "slices": rng.choice([1, 1, 4])}
        if op == "egrad":
            case["out"] = rng.choice(["fp32", "fp32", kind])
        return case
    if op in ("logp", "lgrad"):
        vocab = _width(rng, 200, 262_144)
        n = _log(rng, 1, max(2, min(16_384, 300_000_000 // vocab)))
        case = {"op": op, "n": n, "vocab": vocab, "live": vocab - rng.choice([0, 0, rng.randrange(vocab // 8)]),
                "type": kind, "entropy": rng.random() < 0.5}
        if op == "logp":
            case["top"] = rng.choice([0, 0, 1, 5, rng.randint(2, 16)])
        return case
    hi = _log(rng, 1000, 16_000_000)
    n = max(1, min(_log(rng, 4, 1500), 400_000_000 // max(1, hi // 4)))
    return {"op": op, "list": "ragged", "n": n, "lo": 8, "hi": hi, "type": kind,
            "out": rng.choice(["fp32", kind]), "sizes": rng.randrange(1 << 20)}


# ------------------------------------------------------------------ inputs --

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 29)
    return g


def _zipf(vocab):
    p = 1.0 / (np.arange(vocab) + 2.7)
    return p / p.sum()


def _tokens(n, vocab, g, kind):
    """n token ids below vocab: Zipf ranks, spread over the ids by a multiplier prime to the vocabulary."""
    cdf = torch.from_numpy(np.cumsum(_zipf(vocab))).cuda()
    rank = torch.searchsorted(cdf, torch.rand(n, dtype=torch.float64, device="cuda", generator=g)).clamp_(max=vocab - 1)
    step = next(s for s in range(int(vocab * 0.618) | 1, 2 * vocab + 3, 2) if math.gcd(s, vocab) == 1)
    return (rank * step % vocab).to(getattr(torch, kind))


def _normal(shape, std, g, kind):
    return torch.empty(shape, dtype=TYPES[kind], device="cuda").normal_(0.0, std, generator=g)


def _sizes(c):
    """Elements of each tensor of the list."""
    if c["list"] == "gpt":
        h = HIDDEN
        layer = [h, h, 3 * h * h, 3 * h, h * h, h, h, h, 4 * h * h, 4 * h, 4 * h * h, h]
        return [VOCAB * h, SEQ * h] + c["n"] * layer + [h, h]
    r = random.Random(c["sizes"])
    return [_log(r, c["lo"], c["hi"]) for _ in range(c["n"])]


def _views(c, kind):
    """One flat buffer, as a gradient buffer is, and its consecutive views of the list's sizes."""
    flat = torch.empty(sum(_sizes(c)), dtype=TYPES[kind], device="cuda")
    return flat, list(flat.split(_sizes(c)))


def prepare(case, seed):
    c, g = case, _generator(seed)
    op = c["op"]
    state = {"case": c}
    if op in ("embed", "egrad"):
        state["tokens"] = _tokens(c["n"], c["vocab"] * c["slices"], g, c["ids"])
        state["start"] = c["vocab"] * (c["slices"] // 2)
        state["scale"] = math.sqrt(c["hidden"]) if op == "embed" else 1.0 / 8
        rows = c["vocab"] if op == "embed" else c["n"]
        state["rows"] = _normal((rows, c["hidden"]), 0.02, g, c["type"])
    elif op in ("logp", "lgrad"):
        x = _normal((c["n"], c["vocab"]), 3.0, g, c["type"])
        target = _tokens(c["n"], c["live"], g, "int64")
        lift = 8.0 + 4.0 * torch.rand(c["n"], 1, device="cuda", generator=g)
        x.scatter_add_(1, target[:, None], lift.to(x.dtype))
        x[:, c["live"]:] = -math.inf
        if c["n"] > 32:   # prompt tokens, which have no loss
            target[torch.rand(c["n"], device="cuda", generator=g) < 0.05] = IGNORED
        state.update(logits=x, target=target, scale=1.0 if c["type"] == "bf16" else 1.25)
        if op == "lgrad":
            z = x.double() * state["scale"]
            lse = z.logsumexp(1)
            p = (z - lse[:, None]).exp_()
            state["lse"] = lse.float()
            state["entropy"] = (lse - (p * z.nan_to_num_(neginf=0.0)).sum(1)).float() if c["entropy"] else None
            state["dlogp"] = -torch.rand(c["n"], device="cuda", generator=g)
            state["dentropy"] = 0.01 * torch.rand(c["n"], device="cuda", generator=g) if c["entropy"] else None
    else:
        flat, grads = _views(c, c["type"])
        flat.normal_(0.0, 1.0, generator=g)
        spread = torch.exp(2.0 * torch.randn(len(grads), device="cuda", generator=g) - 5.0)
        torch._foreach_mul_(grads, list(spread.to(flat.dtype)))
        state.update(grads=grads, scale=1.0 / 16, most=0.25)
        if op == "clip":
            state["out"], outs = _views(c, c["out"])
        if own:   # the list of a model's gradient buffers is made once and kept
            state["list"] = _pkg().GradList(grads, out=outs if op == "clip" else None)
    return state


# -------------------------------------------------------------- one pass --

def _inside(tokens, start, vocab):
    ids = tokens.long() - start
    return ids, (ids >= 0) & (ids < vocab)


def _run_plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "embed":
        ids, ok = _inside(s["tokens"], s["start"], c["vocab"])
        rows = s["rows"][torch.where(ok, ids, 0)].float() * s["scale"]
        return torch.where(ok[:, None], rows, 0.0).to(s["rows"].dtype)
    if op == "egrad":
        ids, ok = _inside(s["tokens"], s["start"], c["vocab"])
        grad = torch.zeros(c["vocab"] + 1, c["hidden"], device="cuda")
        grad.index_add_(0, torch.where(ok, ids, c["vocab"]), s["rows"].float())
        return (grad[:-1] * s["scale"]).to(TYPES[c["out"]])
    if op == "logp":
        x = s["logits"].float()
        z = x * s["scale"]
        z = z - z.amax(1, keepdim=True)
        e = z.exp()
        total = e.sum(1, keepdim=True)
        logp = z - total.log()
        ok = s["target"] >= 0
        at = torch.where(ok, s["target"], 0)[:, None]
        out = {"logprobs": torch.where(ok, logp.gather(1, at)[:, 0], 0.0),
               "lse": (x.amax(1, keepdim=True) * s["scale"] + total.log())[:, 0]}
        if c["entropy"]:
            out["entropy"] = -torch.where(e > 0, e / total * logp, 0.0).sum(1)
        if c["top"]:
            out["top_tokens"] = x.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
            out["top_logprobs"] = logp.gather(1, out["top_tokens"])
        return out
    if op == "lgrad":
        logp = s["logits"].float() * s["scale"] - s["lse"][:, None]
        p = logp.exp()
        ok = s["target"] >= 0
        g = torch.where(ok, s["dlogp"], 0.0)[:, None]
        d = -p * g
        if c["entropy"]:
            d = d - torch.where(p > 0, p * (logp + s["entropy"][:, None]) * s["dentropy"][:, None], 0.0)
        d.scatter_add_(1, torch.where(ok, s["target"], 0)[:, None], g)
        return (d * s["scale"]).to(s["logits"].dtype)
    flat = torch.cat(s["grads"]).float() * s["scale"]
    norm = flat.square().sum().sqrt()
    if op == "norm":
        return norm
    s["out"].copy_(flat * (s["most"] / (norm + EPS)).clamp(max=1.0))
    return {"norm": norm, "out": s["out"]}


def _run_own(s):
    c, op, ec = s["case"], s["case"]["op"], _pkg()
    if op == "embed":
        return ec.embed(s["tokens"], s["rows"], scale=s["scale"], vocab_start=s["start"])
    if op == "egrad":
        return ec.embed_grad(s["tokens"], s["rows"], c["vocab"], scale=s["scale"], vocab_start=s["start"],
                             dtype=TYPES[c["out"]])
    if op == "logp":
        r = ec.token_logprobs(s["logits"], s["target"], scale=s["scale"], entropy=c["entropy"], top=c["top"])
        out = {"logprobs": r.logprobs, "lse": r.lse}
        if c["entropy"]:
            out["entropy"] = r.entropy
        if c["top"]:
            out.update(top_tokens=r.top_tokens, top_logprobs=r.top_logprobs)
        return out
    if op == "lgrad":
        return ec.token_logprobs_grad(s["logits"], s["target"], s["lse"], s["dlogp"], scale=s["scale"],
                                      entropy=s["entropy"], dentropy=s["dentropy"])
    if op == "norm":
        return s["list"].norm(grad_scale=s["scale"])
    return {"norm": s["list"].clip(s["most"], grad_scale=s["scale"]), "out": s["out"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------- work, checks --

def _distinct(c):
    """(distinct tokens of the slice, positions in it) to expect among n draws."""
    p = _zipf(c["vocab"] * c["slices"])
    at = np.arange(p.size)
    step = next(s for s in range(int(p.size * 0.618) | 1, 2 * p.size + 3, 2) if math.gcd(s, p.size) == 1)
    ids = at * step % p.size
    start = c["vocab"] * (c["slices"] // 2)
    here = p[(ids >= start) & (ids < start + c["vocab"])]
    return float(np.sum(-np.expm1(c["n"] * np.log1p(-here)))), c["n"] * float(here.sum())


def work(case):
    c, op = case, case["op"]
    if op in ("embed", "egrad"):
        distinct, inside = _distinct(c)
        ids, w = c["n"] * (4 if c["ids"] == "int32" else 8), WIDTH[c["type"]]
        if op == "embed":
            return {"bytes": ids + (distinct + c["n"]) * c["hidden"] * w, "flops": inside * c["hidden"]}
        return {"bytes": ids + inside * c["hidden"] * w + c["vocab"] * c["hidden"] * WIDTH[c["out"]],
                "flops": inside * c["hidden"]}
    if op in ("logp", "lgrad"):
        w, cells = WIDTH[c["type"]], c["n"] * c["vocab"]
        if op == "logp":
            rows = 8 + 4 + 4 + 4 * c["entropy"] + 12 * c["top"]
            return {"bytes": cells * w + c["n"] * rows, "flops": cells * (6 if c["entropy"] else 4)}
        return {"bytes": 2 * cells * w + c["n"] * (16 + 8 * c["entropy"]), "flops": cells * (7 if c["entropy"] else 4)}
    n = sum(_sizes(c))
    if op == "norm":
        return {"bytes": n * WIDTH[c["type"]] + 4, "flops": 3 * n}
    return {"bytes": n * (WIDTH[c["type"]] + WIDTH[c["out"]]) + 4, "flops": 4 * n}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    c, op = case, case["op"]
    if op in ("embed", "egrad"):
        ids = s["tokens"].to(torch.int64) - s["start"]
        here = ((ids >= 0) & (ids < c["vocab"])).nonzero()[:, 0]
        out = torch.zeros(c["n"] if op == "embed" else c["vocab"], c["hidden"], dtype=torch.float64, device="cuda")
        if op == "embed":
            out[here] = s["rows"][ids[here]].double() * s["scale"]
        else:
            out.index_add_(0, ids[here], s["rows"][here].double() * s["scale"])
        return out
    if op in ("logp", "lgrad"):
        z = s["logits"].double() * s["scale"]
        has = (s["target"] >= 0).double()
        one = torch.zeros_like(z).scatter_(1, s["target"].clamp(min=0)[:, None], has[:, None])
        if op == "logp":
            lse = torch.logsumexp(z, 1)
            given = torch.gather(z, 1, s["target"].clamp(min=0)[:, None])[:, 0]
            out = {"logprobs": (given - lse) * has, "lse": lse}
            if c["entropy"]:
                p = torch.exp(z - lse[:, None])
                out["entropy"] = lse - torch.where(p > 0, p * z, 0.0).sum(1)
            if c["top"]:
                order = s["logits"].double().argsort(dim=1, descending=True, stable=True)[:, :c["top"]]
                out.update(top_tokens=order, top_logprobs=z.gather(1, order) - lse[:, None])
            return out
        q = z - s["lse"].double()[:, None]
        weight = (s["dlogp"].double() * has)[:, None]
        p = torch.exp(q)
        d = weight * (one - p)
        if c["entropy"]:
            inner = (q + s["entropy"].double()[:, None]).masked_fill(p == 0, 0.0)
            d -= s["dentropy"].double()[:, None] * p * inner
        return d * s["scale"]
    squares = sum(float(g.double().square().sum()) for g in s["grads"])
    norm = torch.tensor(math.sqrt(squares) * s["scale"], dtype=torch.float64)
    if op == "norm":
        return norm
    by = s["scale"] * min(1.0, s["most"] / (float(norm) + EPS))
    return {"norm": norm, "out": torch.cat([g.double() * by for g in s["grads"]])}
