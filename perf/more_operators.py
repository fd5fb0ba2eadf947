"""The operators of a block between the embedding and the loss, and of its matrices' update, one pass each: their plain
forms in elementary torch operations, and the calls a user makes of the framework.

  ortho     an update orthogonalised by Newton-Schulz products, scaled, alone or added to the decayed weights
  ff        the gated feed-forward: both projections, the activation and the product
  ffgrad    its gradients with respect to the input and both weights, with the projections computed again
  norm      a branch normalised, gated, scaled and added to the residual stream, and the sum normalised for what follows
  normgrad  its gradients with respect to the stream, the branch, the gate and both norms' weights

Updates are a part of low rank with noise around it, as momenta of gradients are. Inputs of the feed-forward are normal,
as a norm leaves them; its weights are normal, divided by the root of their width. The residual stream is wide, with a few
columns an order of magnitude above the others.
"""
import math
import random  # noqa: F401  (draw takes a random.Random)

import torch

own = False

HIDDEN, FFN, LAYERS, SEQ = 2048, 8192, 24, 2048   # the 1.3B-parameter GPT of the engine's benchmark
SMALL = 128                                        # the hidden size of the example's model
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH = {"fp32": 4, "bf16": 2, "fp16": 2}
STEPS, COEFFICIENTS, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, DECAY = 0.02, 0.1
NORM_EPS = 1e-6


def _pkg():
    import __graft_entry__
    return __graft_entry__.load_package()


def listed():
    return [
        # the update of one small matrix, as the example's model has: latency
        {"name": "ortho_128", "op": "ortho", "batch": 1, "rows": SMALL, "cols": SMALL, "type": "bf16", "out": "bf16",
         "base": False},
        # odd tall matrices of a few layers, in fp32
        {"name": "ortho_odd", "op": "ortho", "batch": 5, "rows": 1001, "cols": 777, "type": "fp32", "out": "fp32",
         "base": False},
        # one layer's up projection, its fp32 weights decayed and updated from a bf16 momentum
        {"name": "ortho_up", "op": "ortho", "batch": 1, "rows": FFN, "cols": HIDDEN, "type": "bf16", "out": "fp32",
         "base": True},
        # the square matrices of all layers in one stack
        {"name": "ortho_layers", "op": "ortho", "batch": LAYERS, "rows": HIDDEN, "cols": HIDDEN, "type": "bf16",
         "out": "bf16", "base": False},
        # a single new token of a served sequence
        {"name": "ff_token", "op": "ff", "n": 1, "width": HIDDEN, "inner": FFN, "type": "bf16", "act": "silu"},
        # a training step's micro-batch: eight sequences of 2048 tokens
        {"name": "ff_16k", "op": "ff", "n": 8 * SEQ, "width": HIDDEN, "inner": FFN, "type": "bf16", "act": "silu"},
        # a ragged batch through odd widths, in fp16
        {"name": "ffgrad_777", "op": "ffgrad", "n": 777, "width": 1001, "inner": 1333, "type": "fp16", "act": "gelu_tanh"},
        # the backward pass of four sequences
        {"name": "ffgrad_8k", "op": "ffgrad", "n": 4 * SEQ, "width": HIDDEN, "inner": FFN, "type": "bf16", "act": "silu"},
        # the norms around a block while eight sequences decode
        {"name": "norm_8", "op": "norm", "n": 8, "width": HIDDEN, "type": "bf16", "post": True, "gate": 0},
        # a micro-batch of eight sequences, each with a gate of its own
        {"name": "norm_16k", "op": "norm", "n": 8 * SEQ, "width": HIDDEN, "type": "bf16", "post": True, "gate": 8},
        # odd rows and an odd width in fp32, one gate for all rows, no norm on the branch
        {"name": "normgrad_1023", "op": "normgrad", "n": 1023, "width": 1999, "type": "fp32", "post": False, "gate": 1},
        # the backward pass of the micro-batch
        {"name": "normgrad_16k", "op": "normgrad", "n": 8 * SEQ, "width": HIDDEN, "type": "bf16", "post": True, "gate": 8},
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _width(rng, lo, hi):
    """A size between lo and hi, odd in half of the cases, else 8 past a multiple of 64 or a power of two."""
    n = _log(rng, lo, hi)
    how = rng.random()
    if how < 0.5:
        return n | 1
    return max(lo, n // 64 * 64 + 8) if how < 0.75 else 1 << max(4, n.bit_length() - 1)


def draw(rng):
    op = rng.choice(["ortho", "ortho", "ff", "ff", "ffgrad", "norm", "normgrad"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "ortho":
        rows, cols = _width(rng, 16, 4096), _width(rng, 16, 4096)
        least, most = sorted((rows, cols))
        room = LAYERS * HIDDEN ** 3 / (least * least * most)
        batch = _log(rng, 1, max(1.0, min(32.0, room))) if room > 1 else 1
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "type": kind,
                "out": rng.choice([kind, "fp32"]), "base": rng.random() < 0.4}
    if op in ("ff", "ffgrad"):
        width, inner = _width(rng, 16, 4096), _width(rng, 16, 16_384)
        n = _log(rng, 1, max(2, min(16_384, 4 * SEQ * HIDDEN * FFN // (width * inner))))
        return {"op": op, "n": n, "width": width, "inner": inner, "type": kind,
                "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh"])}
    width = _width(rng, 16, 8192)
    n = _log(rng, 1, max(2, min(32_768, 8 * SEQ * HIDDEN // width)))
    gate = rng.choice([0, 1, n, 4])   # none, one for all rows, one a row, four groups of rows
    n = n // 4 * 4 + 4 if gate == 4 else n
    return {"op": op, "n": n, "width": width, "type": kind, "post": rng.random() < 0.6, "gate": gate}


# ------------------------------------------------------------------ inputs --

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1_000_003 + 41)
    return g


def _normal(shape, std, g, kind="fp32"):
    return torch.empty(shape, dtype=TYPES[kind], device="cuda").normal_(0.0, std, generator=g)


def _stream(c, g):
    """Rows of a residual stream: unit spread, every 97th column ten times that."""
    x = _normal((c["n"], c["width"]), 1.0, g)
    x[:, 5::97] *= 10.0
    return x.to(TYPES[c["type"]])


def prepare(case, seed):
    c, g = case, _generator(seed)
    op, kind = c["op"], c["type"]
    state = {"case": c}
    if op == "ortho":
        b, m, n = c["batch"], c["rows"], c["cols"]
        r = max(1, min(m, n) // 16)
        low = _normal((b, m, r), 1.0, g) @ _normal((b, r, n), 1.0, g) / math.sqrt(r)
        state["update"] = ((low + _normal((b, m, n), 0.2, g)) * 0.01).to(TYPES[kind])
        state["base"] = _normal((b, m, n), 0.02, g, c["out"]) if c["base"] else None
        state["scale"] = math.sqrt(max(1.0, m / n)) * (-LR if c["base"] else 1.0)
        state["keep"] = 1.0 - LR * DECAY
    elif op in ("ff", "ffgrad"):
        k, f = c["width"], c["inner"]
        state["x"] = _normal((c["n"], k), 1.0, g, kind)
        weight = _normal((2 * f, k), 1.0 / math.sqrt(k), g, kind)   # one buffer, as a fused first layer has it
        state["w_gate"], state["w_up"] = weight[:f], weight[f:]
        if op == "ffgrad":
            state["dh"] = _normal((c["n"], f), 0.1, g, kind)
    else:
        n, w = c["n"], c["width"]
        state["residual"] = _stream(c, g)
        state["branch"] = _normal((n, w), 0.5, g, kind)
        state["weight"] = (1.0 + _normal((w,), 0.2, g)).to(TYPES[kind])
        state["branch_weight"] = (0.5 + _normal((w,), 0.1, g)).to(TYPES[kind]) if c["post"] else None
        state["gate"] = _normal((c["gate"], w), 0.7, g, kind) if c["gate"] else None
        state["scale"] = 1.0 / math.sqrt(2 * LAYERS)
        if op == "normgrad":   # residual is the stream behind the sum, and the forward pass left both norms' factors
            root = lambda t: (t.double().square().mean(1) + NORM_EPS).rsqrt().float()   # noqa: E731
            state["rstd"] = root(state["residual"])
            state["branch_rstd"] = root(state["branch"]) if c["post"] else None
            state["dresidual"] = _normal((n, w), 0.1, g, kind)
            state["dnormed"] = _normal((n, w), 0.1, g, kind)
    return state


# -------------------------------------------------------------- one pass --

def _act(g, act):
    """The activation and its derivative."""
    if act == "silu":
        s = 1.0 / (1.0 + (-g).exp())
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "gelu":
        p = 0.5 * (1.0 + (g * math.sqrt(0.5)).erf())
        return g * p, p + g * (-0.5 * g * g).exp() * (0.5 * math.sqrt(2.0 / math.pi))
    r = math.sqrt(2.0 / math.pi)
    t = (r * (g + 0.044715 * g * g * g)).tanh()
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * r * (1.0 + 3 * 0.044715 * g * g)


def _rows_of(gate, n):
    """A gate's rows for each of n rows, which they share evenly in order."""
    return gate.float().repeat_interleave(n // gate.shape[0], 0)


def _run_plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "ortho":
        x = s["update"].float()
        tall = c["rows"] > c["cols"]
        x = x.mT.contiguous() if tall else x
        x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + NS_EPS)
        a, b, k = COEFFICIENTS
        for _ in range(STEPS):
            gram = x @ x.mT.contiguous()
            x = a * x + (b * gram + k * (gram @ gram)) @ x
        x = (x.mT if tall else x) * s["scale"]
        if s["base"] is not None:
            x = s["base"].float() * s["keep"] + x
        return x.to(TYPES[c["out"]]).contiguous()
    if op in ("ff", "ffgrad"):
        x, w1, w2 = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
        g, u = x @ w1.t(), x @ w2.t()
        a, da = _act(g, c["act"])
        if op == "ff":
            return (a * u).to(s["x"].dtype)
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        out = {"dx": dg @ w1 + du @ w2, "dw_gate": dg.t() @ x, "dw_up": du.t() @ x}
        return {k: v.to(s["x"].dtype) for k, v in out.items()}
    n, kind = c["n"], s["residual"].dtype
    r, y, w = s["residual"].float(), s["branch"].float(), s["weight"].float()
    gate = _rows_of(s["gate"], n) if c["gate"] else 1.0
    if op == "norm":
        if c["post"]:
            y = y * (y.square().mean(1, keepdim=True) + NORM_EPS).rsqrt() * s["branch_weight"].float()
        r = r + s["scale"] * gate * y
        rstd = (r.square().mean(1, keepdim=True) + NORM_EPS).rsqrt()
        return {"residual": r.to(kind), "normed": (r * rstd * w).to(kind), "rstd": rstd[:, 0]}
    dz = s["dnormed"].float()
    hat = r * s["rstd"][:, None]
    dhat = dz * w
    d = s["dresidual"].float() + s["rstd"][:, None] * (dhat - hat * (dhat * hat).mean(1, keepdim=True))
    out = {"residual": d.to(kind), "weight": (dz * hat).sum(0)}
    yhat = y * s["branch_rstd"][:, None] if c["post"] else y
    shown = yhat * s["branch_weight"].float() if c["post"] else y
    if c["gate"]:
        out["gate"] = (s["scale"] * d * shown).reshape(c["gate"], n // c["gate"], c["width"]).sum(1)
    dy = s["scale"] * gate * d
    if c["post"]:
        out["branch_weight"] = (dy * yhat).sum(0)
        dy = dy * s["branch_weight"].float()
        dy = s["branch_rstd"][:, None] * (dy - yhat * (dy * yhat).mean(1, keepdim=True))
    out["branch"] = dy.to(kind)
    return out


def _run_own(s):
    c, op, ec = s["case"], s["case"]["op"], _pkg()
    if op == "ortho":
        return ec.orthogonalize(s["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS, scale=s["scale"],
                                base=s["base"], keep=s["keep"], dtype=TYPES[c["out"]])
    if op == "ff":
        return ec.gated_ff(s["x"], s["w_gate"], s["w_up"], activation=c["act"])
    if op == "ffgrad":
        return ec.gated_ff_grad(s["dh"], s["x"], s["w_gate"], s["w_up"], activation=c["act"])._asdict()
    if op == "norm":
        r = ec.residual_norm(s["residual"], s["branch"], gate=s["gate"], scale=s["scale"],
                             branch_weight=s["branch_weight"], weight=s["weight"], eps=NORM_EPS)
        return {"residual": r.residual, "normed": r.normed, "rstd": r.rstd}
    r = ec.residual_norm_grad(s["dresidual"], s["dnormed"], s["residual"], s["branch"], rstd=s["rstd"],
                              branch_rstd=s["branch_rstd"], gate=s["gate"], scale=s["scale"],
                              branch_weight=s["branch_weight"], weight=s["weight"])
    return {k: v for k, v in r._asdict().items() if v is not None}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------- work, checks --

def work(case):
    c, op = case, case["op"]
    w = WIDTH[c["type"]]
    if op == "ortho":
        b, m, n = c["batch"], min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
        cells = b * m * n
        # a step's two symmetric products need half of their entries
        return {"bytes": cells * (w + WIDTH[c["out"]] * (2 if c["base"] else 1)),
                "flops": STEPS * b * (m * m * n + m * m * m + 2 * m * m * n)}
    if op in ("ff", "ffgrad"):
        n, k, f = c["n"], c["width"], c["inner"]
        if op == "ff":
            return {"bytes": (n * k + 2 * f * k + n * f) * w, "flops": 4 * n * k * f}
        return {"bytes": 2 * (n * k + 2 * f * k) * w + n * f * w, "flops": 12 * n * k * f}
    n, k = c["n"], c["width"]
    vectors = k * (1 + c["post"] + c["gate"])
    if op == "norm":
        return {"bytes": 4 * n * k * w + vectors * w + 4 * n, "flops": n * k * (5 + 4 * c["post"])}
    return {"bytes": 6 * n * k * w + vectors * (w + 4) + 4 * n * (1 + c["post"]), "flops": n * k * (9 + 9 * c["post"])}


def exact(case, seed):
    """The definitions in 64 bits; gradients by differentiation of the forward formulas."""
    s = prepare(case, seed)
    c, op = case, case["op"]
    if op == "ortho":
        x = s["update"].double()
        x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + NS_EPS)
        tall = c["rows"] > c["cols"]
        a, b, k = COEFFICIENTS
        out = []
        for one in x:   # the steps' polynomials of the Gram matrix commute: their product, applied once
            side = min(one.shape)
            gram = one.t() @ one if tall else one @ one.t()
            eye = torch.eye(side, dtype=torch.float64, device=one.device)
            total = eye
            for _ in range(STEPS):
                p = a * eye + gram @ (b * eye + k * gram)
                total, gram = p @ total, p @ gram @ p
            out.append(one @ total if tall else total @ one)
        x = torch.stack(out) * s["scale"]
        return x if s["base"] is None else torch.add(x, s["base"].double(), alpha=s["keep"])
    if op in ("ff", "ffgrad"):
        x, w1, w2 = (s[k].double().requires_grad_() for k in ("x", "w_gate", "w_up"))
        with torch.set_grad_enabled(op == "ffgrad"):
            g = torch.matmul(x, w1.t())
            g = torch.nn.functional.silu(g) if c["act"] == "silu" else \
                torch.nn.functional.gelu(g, approximate="tanh" if c["act"] == "gelu_tanh" else "none")
            h = g * torch.matmul(x, w2.t())
        if op == "ff":
            return h
        return dict(zip(("dx", "dw_gate", "dw_up"), torch.autograd.grad(h, (x, w1, w2), s["dh"].double())))
    n, w = c["n"], c["width"]
    r, y, wt = (s[k].double().requires_grad_() for k in ("residual", "branch", "weight"))
    bw = s["branch_weight"].double().requires_grad_() if c["post"] else None
    gate = s["gate"].double().requires_grad_() if c["gate"] else None

    def shown(factor):
        v = y if bw is None else y * factor * bw
        if gate is not None:
            v = (v.view(c["gate"], -1, w) * gate[:, None]).view(n, w)
        return v * s["scale"]

    if op == "norm":
        with torch.no_grad():
            total = r + shown(torch.rsqrt(torch.mean(y * y, 1, keepdim=True) + NORM_EPS))
            rstd = torch.rsqrt(torch.mean(total * total, 1, keepdim=True) + NORM_EPS)
            return {"residual": total, "normed": total * rstd * wt, "rstd": rstd[:, 0]}
    # a norm's factor is differentiated too, at the value that the forward pass left
    factor = lambda t, root: root.double()[:, None] * torch.rsqrt(   # noqa: E731
        1.0 + ((t * t).mean(1, keepdim=True) - (t * t).mean(1, keepdim=True).detach()) * root.double()[:, None] ** 2)
    normed = r * factor(r, s["rstd"]) * wt
    d, dwt = torch.autograd.grad(normed, (r, wt), s["dnormed"].double())
    d = d + s["dresidual"].double()
    out = {"residual": d, "weight": dwt}
    names = {"branch": y, "gate": gate, "branch_weight": bw}
    names = {k: v for k, v in names.items() if v is not None}
    total = shown(factor(y, s["branch_rstd"]) if c["post"] else None)
    out.update(zip(names, torch.autograd.grad(total, list(names.values()), d)))
    return out
