"""Performance cases of the operators between a language model's layers, before its update and behind its logits.

  norm        root-mean-square norm of x (+ the residual stream), also with an output in 8 bits with scales
  norm_grad   its gradients with respect to input and weight
  clip        global norm of a list of gradients, and the gradients scaled down to a limit
  sample      a token per row of logits from given random numbers: temperature, top-k, top-p, min-p

`run` is one call of one of them. Where `own` is false it is the same mathematics in elementary torch operations: in fp32 and rounded
once at the end, or in fp64 where a token depends on which side of a border a sum falls.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
E4M3_MAX = 448.0
LEAST_SCALE = 2.0 ** -126


def _norm(name, rows, width, dtype, residual, out="same", block=0, weight="same"):
    """block: columns per scale of an e4m3 output, 0 for one per row. weight: "same" type as x, or "fp32"."""
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "out": out, "block": block, "weight": weight}


def _norm_grad(name, rows, width, dtype, residual, weight="same"):
    return {"name": name, "op": "norm_grad", "rows": rows, "width": width, "dtype": dtype, "residual": residual, "weight": weight}


def _clip(name, kind, count, size, dtype, over):
    """kind: "equal" tensors of `size` elements, or "ragged" ones of 1 to `size`, side by side in one buffer per type; dtype "mixed": every
    third one fp32. over: the norm is over the limit, and results go to other buffers; otherwise it is under it, in place."""
    return {"name": name, "op": "clip", "kind": kind, "count": count, "size": size, "dtype": dtype, "over": over}


def _sample(name, rows, vocab, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False, masked=0.0):
    """per_row: every row has its own four numbers (the given ones or others, and one row in eight is greedy)."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "temperature": temperature, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "per_row": per_row, "masked": masked}


def listed():
    return [
        # one token of one sequence: latency
        _norm("norm_token", 1, 4096, "bf16", True),
        # between two layers of a training step: 32 sequences of 2048 tokens, with the residual stream
        _norm("norm_step", 65536, 1024, "bf16", True, weight="fp32"),
        # the same in front of an 8-bit product: a scale for each 128 columns
        _norm("norm_e4m3", 8192, 4096, "bf16", True, out="e4m3", block=128),
        # a small fp32 model with odd sizes
        _norm_grad("norm_grad_odd", 1000, 203, "fp32", False),
        # the backward end of norm_step: a gradient arrives at the residual stream as well
        _norm_grad("norm_grad_step", 65536, 1024, "bf16", True, weight="fp32"),
        # the five layers of the 5 x 1024 network
        _clip("clip_5x1024", "equal", 5, 1024 * 1024, "fp32", True),
        # many small tensors of all sizes, vectors in fp32 among matrices in bf16, as one bucket per type
        _clip("clip_ragged", "ragged", 300, 200000, "mixed", True),
        # the eight layers of the 8 x 4096 network; most steps are under the limit
        _clip("clip_8x4096", "equal", 8, 4096 * 4096, "bf16", False),
        # a single answer: latency
        _sample("sample_one", 1, 32768, "fp32", temperature=0.75, top_k=50, top_p=0.9375),
        # a few requests with their own settings over an odd vocabulary, a third of it masked by a grammar
        _sample("sample_odd", 33, 10007, "fp32", temperature=0.875, top_k=40, min_p=0.0625, per_row=True, masked=0.3),
        # a full serving batch, nucleus sampling over the whole vocabulary
        _sample("sample_batch", 256, 65536, "bf16", top_p=0.9375),
        # rollouts for policy gradients: the model's own distribution, with log probabilities
        _sample("sample_rollout", 1024, 65536, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "clip", "clip", "sample", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op in ("norm", "norm_grad"):
        while True:
            r, w = _log(rng, 1, 65536), _log(rng, 16, 16384)
            if r * w <= (1 << 26 if dtype == "bf16" else 1 << 25):
                break
        w = w if rng.random() < 0.4 else -(-w // 64) * 64
        weight, residual = rng.choice(["same", "fp32"]), rng.random() < 0.5
        if op == "norm":
            c = _norm("", r, w, dtype, residual, rng.choice(["same", "same", "e4m3"]), rng.choice([0, 128]), weight)
            c["block"] = c["block"] if c["out"] == "e4m3" else 0
        else:
            c = _norm_grad("", r, w, dtype, residual, weight)
    elif op == "clip":
        kind = rng.choice(["equal", "ragged"])
        count = _log(rng, 1, 600)
        size = _log(rng, 64, min(1 << 24, (1 << 26) // count))
        c = _clip("", kind, count, size, rng.choice([dtype, "mixed"]), rng.random() < 0.6)
    else:
        k, p, m = rng.choice([0, 0, 1, 20, 50, 400]), rng.choice([1.0, 1.0, 0.5, 0.9375, 0.984375]), rng.choice([0.0, 0.0, 0.03125, 0.125])
        per_row = rng.random() < 0.4
        while True:
            r, v = _log(rng, 1, 2048), _log(rng, 64, 262144)
            if r * v <= (1 << 26 if not (k or per_row) and p == 1.0 and dtype == "bf16" else 1 << 24):
                break
        c = _sample("", r, v, dtype, rng.choice([0.0, 0.5, 0.75, 1.0, 1.0, 1.25]), k, p, m, per_row, rng.choice([0.0, 0.0, 0.3, 0.9]))
    return {k: v for k, v in c.items() if k != "name"}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _sizes(case):
    if case["kind"] == "equal":
        return [case["size"]] * case["count"]
    r = random.Random(case["count"] * 1000003 + case["size"])
    return [_log(r, 1, case["size"]) for _ in range(case["count"])]


def _types(case):
    if case["dtype"] == "mixed":
        return ["fp32" if i % 3 == 0 else "bf16" for i in range(case["count"])]
    return [case["dtype"]] * case["count"]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    if op in ("norm", "norm_grad"):
        r, w, dtype = case["rows"], case["width"], DTYPE[case["dtype"]]
        wt = dtype if case["weight"] == "same" else torch.float32
        s = {"op": op, "weight": (1 + 0.2 * randn(w)).to(wt)}
        # rows of different sizes, and a few columns that stand out, as a residual stream has them
        columns = 1 + 8 * (rand(w) < 0.01)
        stream = randn(r, w) * (0.5 + 2 * rand(r, 1)) * columns
        if op == "norm":
            s["x"] = (randn(r, w) * 0.5 if case["residual"] else stream).to(dtype)
            s["residual"] = stream.to(dtype) if case["residual"] else None
            s["e4m3"], s["block"] = case["out"] == "e4m3", case["block"]
            return s
        s["total"] = stream.to(dtype)
        s["dy"] = (randn(r, w) * 1e-3 * (0.2 + rand(r, 1))).to(dtype)
        s["dtotal"] = (randn(r, w) * 1e-3).to(dtype) if case["residual"] else None
        return s
    if op == "clip":
        sizes, types = _sizes(case), _types(case)
        s = {"op": op, "flat": [], "out": [], "grads": [None] * len(sizes), "outs": [None] * len(sizes)}
        squares = 0.0
        for t in ("bf16", "fp32"):
            mine = [i for i, x in enumerate(types) if x == t]
            if not mine:
                continue
            n = sum(sizes[i] for i in mine)
            flat = (randn(n) * 1e-3).to(DTYPE[t])
            out = torch.empty_like(flat) if case["over"] else flat
            for x, views in ((flat, s["grads"]), (out, s["outs"])):
                at = 0
                for i in mine:
                    views[i] = x[at:at + sizes[i]]
                    at += sizes[i]
            s["flat"].append(flat)
            s["out"].append(out)
            squares += float(flat.double().square().sum())
        s["over"] = case["over"]
        s["max_norm"] = float(np.float32(math.sqrt(squares) * (0.375 if case["over"] else 2.0)))
        return s
    r, v = case["rows"], case["vocab"]
    x = randn(r, v) * 2.5
    # a trained model: some continuations stand out of the rest by 2 to 12
    likely = torch.randint(0, v, (r, 24), device="cuda", generator=g)
    x.scatter_add_(1, likely, 2 + 10 * rand(r, 24) ** 3)
    if case["masked"]:
        mask = rand(r, v) < case["masked"]
        mask.scatter_(1, likely[:, :1], False)
        x.masked_fill_(mask, -math.inf)
    s = {"op": op, "logits": x.to(DTYPE[case["dtype"]]), "u": rand(r), "temperature": case["temperature"], "top_k": case["top_k"], "top_p": case["top_p"],
         "min_p": case["min_p"]}
    if case["per_row"]:
        pick = lambda values, t: torch.tensor(values, device="cuda", dtype=t)[torch.randint(0, len(values), (r,), device="cuda", generator=g)]  # noqa: E731
        t = case["temperature"]
        s["temperature"] = pick([t, t, t, 0.5, 0.75, 1.0, 1.125, 0.0], torch.float32)
        s["top_k"] = pick([case["top_k"], case["top_k"], 0, 5, 100], torch.int32)
        s["top_p"] = pick([case["top_p"], case["top_p"], 1.0, 0.75], torch.float32)
        s["min_p"] = pick([case["min_p"], case["min_p"], 0.0, 0.125], torch.float32)
    return s


def _plain_norm(s):
    t = s["x"]
    if s["residual"] is not None:
        t = (t.float() + s["residual"].float()).to(t.dtype)
    f = t.float()
    y = f * (f.square().mean(1, keepdim=True) + EPS).rsqrt() * s["weight"].float()
    if not s["e4m3"]:
        y = y.to(t.dtype)
        return y if s["residual"] is None else (y, t)
    rows, width = y.shape
    block = s["block"] or width
    blocks = -(-width // block)
    padded = torch.zeros(rows, blocks * block, device=y.device)
    padded[:, :width] = y
    padded = padded.view(rows, blocks, block)
    scale = (padded.abs().amax(2) / E4M3_MAX).clamp(min=LEAST_SCALE)
    q = (padded / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(rows, -1)[:, :width].to(torch.float8_e4m3fn)
    return (q, scale) if s["residual"] is None else (q, scale, t)


def _plain_norm_grad(s):
    t, dy, w = s["total"].float(), s["dy"].float(), s["weight"].float()
    r = (t.square().mean(1, keepdim=True) + EPS).rsqrt()
    n = t * r
    g = dy * w
    dx = r * (g - n * (g * n).mean(1, keepdim=True))
    if s["dtotal"] is not None:
        dx = dx + s["dtotal"].float()
    return dx.to(s["total"].dtype), (dy * n).sum(0).to(s["weight"].dtype)


def _plain_clip(s):
    squares = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]])
    norm = squares.sum().sqrt()
    factor = (s["max_norm"] / norm).clamp(max=1.0).float()
    [y.copy_((x.float() * factor).to(x.dtype)) for x, y in zip(s["grads"], s["outs"])]
    return [norm.float()] + s["out"]


def _column(v, like):
    return v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((like.shape[0], 1), float(v), device=like.device, dtype=torch.float64)


def _plain_sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(vocab, device=x.device)
    temperature, top_k, top_p, min_p = (_column(s[k], x) for k in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature <= 0
    first = x.argmax(1, keepdim=True)
    y = (x.double() - x.gather(1, first).double()) / torch.where(greedy, 1.0, temperature)
    w = y.exp()
    if isinstance(s["top_k"], torch.Tensor) or s["top_k"] > 0 or s["top_p"] < 1:
        order = x.sort(dim=1, descending=True, stable=True).indices
        sorted_w = w.gather(1, order)
        among = (at < top_k) | (top_k <= 0)
        sorted_w = torch.where(among, sorted_w, 0.0)
        before = sorted_w.cumsum(1) - sorted_w
        keep = among & ((before < top_p * sorted_w.sum(1, keepdim=True)) | (top_p >= 1)) & (sorted_w >= min_p) | (at == 0)
        kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sorted_w, 0.0))
    else:
        kept = torch.where((w >= min_p) | (at == first), w, 0.0)
    cum = kept.cumsum(1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    token = torch.minimum(token, torch.where(kept > 0, at, -1).amax(1, keepdim=True))
    token = torch.where(greedy, first, token)
    logprob = torch.where(greedy, 0.0, y.gather(1, token) - total.log())
    return token[:, 0], logprob[:, 0].float()


def run(s):
    op = s["op"]
    if not own:
        return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "clip": _plain_clip, "sample": _plain_sample}[op](s)
    from tbb_test_b200 import lm
    if op == "norm":
        if s["e4m3"]:
            return lm.norm_e4m3(s["x"], s["weight"], residual=s["residual"], eps=EPS, block=s["block"])
        return lm.norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    if op == "norm_grad":
        return lm.norm_grad(s["dy"], s["total"], s["weight"], dtotal=s["dtotal"], eps=EPS)
    if op == "clip":
        norm = lm.clip(s["grads"], s["max_norm"], out=s["outs"] if s["over"] else None)
        return [norm] + s["out"]
    return lm.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], logprob=True)


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        r, w, e = case["rows"], case["width"], 2 if case["dtype"] == "bf16" else 4
        we = e if case["weight"] == "same" else 4
        if op == "norm_grad":  # dy and the sum read, dx written; the weight read and its gradient written
            return {"bytes": r * w * e * (3 + case["residual"]) + 2 * w * we, "flops": 12 * r * w}
        out = e if case["out"] == "same" else 1
        scales = 0 if case["out"] == "same" else 4 * r * -(-w // (case["block"] or w))
        return {"bytes": r * w * (e * (1 + 2 * case["residual"]) + out) + w * we + scales, "flops": 5 * r * w}
    if op == "clip":
        n = sum(z * (4 if t == "fp32" else 2) for z, t in zip(_sizes(case), _types(case)))
        return {"bytes": n * (2 if case["over"] else 1) + 4, "flops": 3 * sum(_sizes(case))}
    r, v, e = case["rows"], case["vocab"], 2 if case["dtype"] == "bf16" else 4
    return {"bytes": r * (v * e + 16) + (16 * r if case["per_row"] else 0), "flops": 4 * r * v}


def _exact_row(x, u, temperature, top_k, top_p, min_p):
    """(token, log probability) of one row, float64 on the host."""
    best = int(np.argmax(x))
    if temperature <= 0:
        return best, 0.0
    with np.errstate(under="ignore"):
        w = np.exp((x - x[best]) / temperature)
    if top_k > 0 or top_p < 1:
        some = np.lexsort((np.arange(len(x)), -x))[:top_k if top_k > 0 else None]
        n = len(some)
        if top_p < 1:
            sums = np.cumsum(w[some])
            n = min(n, max(1, int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1))
        kept = np.sort(some[:max(1, min(n, int((w[some[:n]] >= min_p).sum())))])
    else:
        kept = np.flatnonzero((w >= min_p) | (np.arange(len(x)) == best))
    sums = np.cumsum(w[kept])
    i = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(kept) - 1)
    while i and w[kept[i]] == 0:
        i -= 1
    return kept[i], math.log(w[kept[i]] / sums[-1])


def exact(case, seed):
    """The outputs from the definitions, in 64 bits."""
    s = prepare(case, seed)
    op = s["op"]
    if op == "norm":
        x = s["x"].double()
        if s["residual"] is not None:
            x = (x + s["residual"].double()).to(s["x"].dtype).double()
        y = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / x.shape[1] + EPS) * s["weight"].double()
        total = [] if s["residual"] is None else [x]
        if not s["e4m3"]:
            return y if not total else (y, x)
        block = s["block"] or x.shape[1]
        parts = y.split(block, 1)
        scales = torch.stack([torch.linalg.vector_norm(p, math.inf, dim=1) / E4M3_MAX for p in parts], 1).clamp(min=LEAST_SCALE)
        q = []
        for i, p in enumerate(parts):
            v = p / scales[:, i:i + 1]
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)  # three bits behind the leading one, subnormals below 2^-6
            q.append(torch.round(v / step) * step)
        return (torch.cat(q, 1), scales, *total)
    if op == "norm_grad":
        t, w = s["total"].double().requires_grad_(), s["weight"].double().requires_grad_()
        y = t / torch.sqrt((t ** 2).mean(1, keepdim=True) + EPS) * w
        dt, dw = torch.autograd.grad(y, (t, w), s["dy"].double())
        return dt if s["dtotal"] is None else dt + s["dtotal"].double(), dw
    if op == "clip":
        norm = math.sqrt(sum(float(torch.dot(x.double(), x.double())) for x in s["flat"]))
        factor = min(1.0, s["max_norm"] / norm)
        return [norm] + [x.double() * factor for x in s["flat"]]
    x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    rows = len(x)
    every = [v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, float(v)) for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    got = [_exact_row(x[i], u[i], every[0][i], int(every[1][i]), every[2][i], every[3][i]) for i in range(rows)]
    return torch.tensor([int(t) for t, _ in got]), torch.tensor([p for _, p in got], dtype=torch.float64)
