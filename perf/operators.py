"""Performance cases of the operators a language model's training step needs around the network's own layers.

  embed       rows of a table by token number, scaled          (input of the network)
  embed_grad  the table's gradient, summed by sorted tokens     (end of the backward pass)
  xent        softmax cross entropy behind a vocabulary-wide    (output: loss, and the gradients of the layer's
              linear layer, logits never kept whole              input and weights where `grad` is set)
  muon        momentum and Newton-Schulz orthogonalised update  (weights of the layers between)

`run` is one call of one of them. Where `own` is false it is the same mathematics in elementary torch operations, in
fp32 whatever the inputs' type and rounded once at the end.

A token or target outside [0, vocab) is padding: an embedding row of zeros, no gradient, no loss.
"""
import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
NS = (3.4445, -4.7750, 2.0315)  # the quintic's coefficients: X <- (a + b XX' + c (XX')^2) X
EPS = 1e-7


def _embed(name, tokens, width, vocab, dtype, op="embed", **kw):
    return {"name": name, "op": op, "tokens": tokens, "width": width, "vocab": vocab, "dtype": dtype, "padding": 0.02, **kw}


def _xent(name, rows, width, vocab, dtype, grad, padding=0.1):
    return {"name": name, "op": "xent", "rows": rows, "width": width, "vocab": vocab, "dtype": dtype, "grad": grad, "padding": padding}


def _muon(name, count, rows, cols, grad_dtype, copy, nesterov=True):
    return {"name": name, "op": "muon", "count": count, "rows": rows, "cols": cols, "dtype": grad_dtype, "copy": copy, "nesterov": nesterov}


def listed():
    return [
        # a small interactive batch: one look-up of a few hundred tokens, where the call's latency counts
        _embed("embed_small", 256, 512, 32768, "bf16"),
        # the input of a training step: 32 sequences of 2048 tokens
        _embed("embed_step", 65536, 1024, 65536, "bf16"),
        # a small fp32 model with odd sizes: few tokens, rows that are not whole 16-byte pieces
        _embed("embed_grad_odd", 1000, 203, 10007, "fp32", op="embed_grad"),
        # the backward end of the step above; word frequencies fall as 1 / rank, so some tokens come thousands of times
        _embed("embed_grad_step", 65536, 1024, 65536, "bf16", op="embed_grad"),
        # evaluation of a few positions on an odd vocabulary: reading the weights once is the work
        _xent("xent_eval_small", 96, 512, 10007, "bf16", False),
        # a small training step in fp32, the framework's default precision
        _xent("xent_step_fp32", 1024, 512, 8192, "fp32", True),
        # fine-tuning: more than half of the positions are prompt and carry no loss
        _xent("xent_tune", 4096, 1024, 32768, "bf16", True, padding=0.6),
        # the largest training step: 8192 positions over a vocabulary of 64 Ki, layers of 2048
        _xent("xent_step", 8192, 2048, 65536, "bf16", True),
        # one small layer, where launches and latency are the time
        _muon("muon_small", 1, 256, 256, "fp32", False),
        # all five layers of the 5 x 1024 network
        _muon("muon_5x1024", 5, 1024, 1024, "fp32", True),
        # three tall layers with odd sizes, bf16 gradients
        _muon("muon_ragged", 3, 2001, 515, "bf16", False, nesterov=False),
        # the eight layers of the 8 x 4096 network, bf16 gradients and the bf16 operand copy
        _muon("muon_8x4096", 8, 4096, 4096, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "xent", "xent", "muon", "muon"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("embed", "embed_grad"):
        while True:
            n, d, v = _log(rng, 1, 131072), _log(rng, 48, 4096), _log(rng, 200, 131072)
            if n * d <= 1 << 27 and v * d <= 1 << 27:
                break
        d = d if rng.random() < 0.4 else -(-d // 64) * 64
        return _unnamed(dict(_embed("", n, d, v, dtype, op=op), padding=rng.choice([0.0, 0.02, 0.3])))
    if op == "xent":
        top = 8192 * 2048 * 65536 // (1 if dtype == "bf16" else 8)
        while True:
            r, f, v = _log(rng, 1, 8192), _log(rng, 48, 4096), _log(rng, 200, 131072)
            if r * f * v <= top and v * f <= 1 << 28:
                break
        f = f if rng.random() < 0.4 else -(-f // 64) * 64
        return _unnamed(_xent("", r, f, v, dtype, rng.random() < 0.75, rng.choice([0.0, 0.1, 0.6])))
    while True:
        k, m, n = rng.randint(1, 8), _log(rng, 16, 4096), _log(rng, 16, 4096)
        if max(m, n) <= 32 * min(m, n):
            break
    m, n = (m, n) if rng.random() < 0.4 else (-(-m // 64) * 64, -(-n // 64) * 64)
    return _unnamed(_muon("", k, m, n, dtype, rng.random() < 0.5, rng.random() < 0.5))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _tokens(g, n, vocab, padding):
    """Token numbers whose frequency falls as 1 / rank, the ranks spread over the vocabulary; a share of -1, never the first."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    t = torch.exp(u * math.log(vocab + 1)).long().sub_(1).clamp_(0, vocab - 1)
    t = t * 2654435761 % vocab
    pad = torch.rand(n, device="cuda", generator=g) < padding
    pad[0] = False
    return torch.where(pad, torch.full_like(t, -1), t)


def prepare(case, seed):
    g = _gen(seed)
    op, dtype = case["op"], DTYPE[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if op in ("embed", "embed_grad"):
        n, d, v = case["tokens"], case["width"], case["vocab"]
        s = {"op": op, "tokens": _tokens(g, n, v, case["padding"]).int(), "vocab": v, "scale": d ** 0.5 if op == "embed" else 1.0}
        s["x"] = (randn(v, d) * d ** -0.5 if op == "embed" else randn(n, d) * (1e-3 * torch.rand(n, 1, device="cuda", generator=g))).to(dtype)
        return s
    if op == "xent":
        r, f, v = case["rows"], case["width"], case["vocab"]
        t = _tokens(g, r, v, case["padding"])
        w = (randn(v, f) * (2.0 * f ** -0.5)).to(dtype)
        # a half-trained model: the target's logit stands out by 0 to 12
        h = randn(r, f) + w[t.clamp(0)].float() * (3.0 * torch.rand(r, 1, device="cuda", generator=g))
        return {"op": op, "h": h.to(dtype), "w": w, "targets": t, "scale": 1.0 / r, "grad": case["grad"]}
    k, m, n = case["count"], case["rows"], case["cols"]
    b = 512  # gradients as they come from a batch: dz' a, activations behind a ReLU

    def grad():
        return torch.baddbmm(torch.zeros(1, 1, 1, device="cuda"), randn(k, m, b), randn(k, b, n).relu_(), beta=0, alpha=1.0 / b)

    w = (torch.rand(k, m, n, device="cuda", generator=g) * 2 - 1) * n ** -0.5
    return {"op": op, "w": w, "momentum": grad() * 4, "grad": grad().to(dtype), "copy": torch.empty(k, m, n, dtype=torch.bfloat16, device="cuda") if case["copy"] else None,
            "nesterov": case["nesterov"], "lr": 2e-3, "mu": 0.95, "decay": 0.1, "scale": 0.2 * max(m, n) ** 0.5}


def _plain_embed(s):
    t, v = s["tokens"].long(), s["vocab"]
    ok = ((t >= 0) & (t < v))[:, None]
    return torch.where(ok, s["x"].float()[t.clamp(0, v - 1)] * s["scale"], 0.0).to(s["x"].dtype)


def _plain_embed_grad(s):
    t, v = s["tokens"].long(), s["vocab"]
    ok = ((t >= 0) & (t < v))[:, None]
    rows = torch.where(ok, s["x"].float() * s["scale"], 0.0)
    return torch.zeros(v, rows.shape[1], device=rows.device).index_add_(0, t.clamp(0, v - 1), rows).to(s["x"].dtype)


def _plain_xent(s):
    h, w, t = s["h"].float(), s["w"].float(), s["targets"]
    v = w.shape[0]
    ok, at = (t >= 0) & (t < v), t.clamp(0, v - 1)[:, None]
    x = h @ w.T
    top = x.amax(1, keepdim=True)
    target = x.gather(1, at)
    p = x.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = torch.where(ok, (top + total.log() - target)[:, 0], 0.0)
    if not s["grad"]:
        return loss
    p /= total
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=p.dtype))
    p *= torch.where(ok, s["scale"], 0.0)[:, None]
    return loss, (p @ w).to(s["h"].dtype), (p.T @ h).to(s["w"].dtype)


def _muon_math(w, m, g, s):
    """New (weights, momentum), in the type of w."""
    m = m * s["mu"] + g
    x = g + m * s["mu"] if s["nesterov"] else m
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    tall = x.shape[1] > x.shape[2]
    x = x.mT if tall else x
    a, b, c = NS
    for _ in range(5):
        y = x @ x.mT
        x = a * x + (b * y + c * (y @ y)) @ x
    x = x.mT if tall else x
    return w * (1 - s["lr"] * s["decay"]) - x * (s["lr"] * s["scale"]), m


def _plain_muon(s):
    w, m = _muon_math(s["w"], s["momentum"], s["grad"].float(), s)
    s["w"].copy_(w)
    s["momentum"].copy_(m)
    if s["copy"] is None:
        return s["w"], s["momentum"]
    return s["w"], s["momentum"], s["copy"].copy_(w)


def run(s):
    op = s["op"]
    if not own:
        return {"embed": _plain_embed, "embed_grad": _plain_embed_grad, "xent": _plain_xent, "muon": _plain_muon}[op](s)
    from tbb_test_b200 import lm
    if op == "embed":
        return lm.embed(s["tokens"], s["x"], scale=s["scale"])
    if op == "embed_grad":
        return lm.embed_grad(s["tokens"], s["x"], s["vocab"], scale=s["scale"])
    if op == "xent":
        return lm.xent(s["h"], s["w"], s["targets"], scale=s["scale"], grad=s["grad"])
    lm.muon(s["w"], s["momentum"], s["grad"], lr=s["lr"], momentum=s["mu"], nesterov=s["nesterov"], weight_decay=s["decay"],
            scale=s["scale"], eps=EPS, copy=s["copy"])
    return (s["w"], s["momentum"]) if s["copy"] is None else (s["w"], s["momentum"], s["copy"])


def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    op = case["op"]
    if op == "embed":  # the rows that come, each read once, and the output
        return {"bytes": case["tokens"] * (case["width"] * 2 * e + 4), "flops": case["tokens"] * case["width"]}
    if op == "embed_grad":
        return {"bytes": case["tokens"] * (case["width"] * e + 4) + case["vocab"] * case["width"] * e, "flops": case["tokens"] * case["width"]}
    if op == "xent":  # positions without a target need no logits
        r, f, v = case["rows"] * (1 - case["padding"]), case["width"], case["vocab"]
        io = (r + v) * f * e
        if not case["grad"]:
            return {"bytes": io + case["rows"] * 12, "flops": 2 * r * f * v}
        return {"bytes": io + (case["rows"] + v) * f * e + case["rows"] * 12, "flops": 6 * r * f * v}
    k, a, b = case["count"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # weights and momentum read and written, the gradient read; a symmetric product needs half of its elements
    return {"bytes": k * a * b * (16 + e + (2 if case["copy"] else 0)), "flops": 5 * k * (a * a * b + a * a * a + 2 * a * a * b)}


def exact(case, seed):
    """The outputs from the definitions, in 64 bits."""
    s = prepare(case, seed)
    op = s["op"]
    if op in ("embed", "embed_grad"):
        t, x = s["tokens"].tolist(), s["x"].double()
        keep = torch.tensor([i for i, v in enumerate(t) if 0 <= v < s["vocab"]], device="cuda", dtype=torch.long)
        at = s["tokens"].long()[keep]
        if op == "embed":
            out = torch.zeros(len(t), x.shape[1], device="cuda", dtype=torch.float64)
            out[keep] = x[at] * s["scale"]
            return out
        out = torch.zeros(s["vocab"], x.shape[1], device="cuda", dtype=torch.float64)
        order = torch.argsort(at)
        at, rows = at[order], x[keep][order] * s["scale"]
        bounds = torch.searchsorted(at, torch.arange(s["vocab"] + 1, device="cuda"))
        some = (bounds[1:] > bounds[:-1]).nonzero()[:, 0]
        for v, i, j in zip(some.tolist(), bounds[some].tolist(), bounds[some + 1].tolist()):
            out[v] = rows[i:j].sum(0)
        return out
    if op == "xent":
        h, w, t = s["h"].double(), s["w"].double(), s["targets"]
        r, v = h.shape[0], w.shape[0]
        loss = torch.zeros(r, device="cuda", dtype=torch.float64)
        dh, dw = torch.zeros_like(h), torch.zeros_like(w)
        keep = ((t >= 0) & (t < v)).nonzero()[:, 0]
        for rows in keep.split(1024):
            x = h[rows] @ w.T
            lse = torch.logsumexp(x, 1)
            loss[rows] = lse - x[torch.arange(len(rows), device="cuda"), t[rows]]
            if s["grad"]:
                d = torch.exp(x - lse[:, None])
                d[torch.arange(len(rows), device="cuda"), t[rows]] -= 1.0
                d *= s["scale"]
                dh[rows] = d @ w
                dw += d.T @ h[rows]
        return (loss, dh, dw) if s["grad"] else loss
    new_w, new_m = [], []
    for w, m, g in zip(s["w"].double(), s["momentum"].double(), s["grad"].double()):
        m = s["mu"] * m + g
        u = g + s["mu"] * m if s["nesterov"] else m
        x = u / (torch.linalg.norm(u) + EPS)
        for _ in range(5):
            if x.shape[0] <= x.shape[1]:
                p = x @ x.T
                x = NS[0] * x + NS[1] * (p @ x) + NS[2] * (p @ (p @ x))
            else:
                p = x.T @ x
                x = NS[0] * x + NS[1] * (x @ p) + NS[2] * ((x @ p) @ p)
        new_w.append((1 - s["lr"] * s["decay"]) * w - s["lr"] * s["scale"] * x)
        new_m.append(m)
    w, m = torch.stack(new_w), torch.stack(new_m)
    return (w, m) if s["copy"] is None else (w, m, w)
