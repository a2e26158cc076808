"""Tokens drawn from logits (tbb_test_b200.lm.sample) against a plain implementation in 64 bits on the host.

Tokens have to be equal: weights and sums are in fp64 on both sides, so that they could differ only where u or top_p falls within rounding (1e-12 of the whole)
of a step of the running sum; the oracle says how near it came, and no row here may come that near unless both sums are exact. Log probabilities are rounded to
fp32, half a step; the whole weight in them may be a sum of fp32 weights, off by 1.5e-7 (the power of two) + 2e-8 (its argument) + 3 * 2^-24 (a sum of eight) =
3.5e-7 of itself, and the logarithm by as much."""
import ctypes as ct
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def oracle_row(x, u, t, k, p, m):
    """(token, log probability, distance of u and top_p from the nearest step as a share of the whole) of one row, from the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, 0.0, 1.0
    order = sorted(range(len(x)), key=lambda i: (-x[i], i)) if len(x) < 50 else list(np.lexsort((np.arange(len(x)), -x)))
    top = x[order[0]]
    if not t > 0 or k == 1 or p <= 0 or m > 1:
        return order[0], 0.0, 1.0
    t = min(t, float(np.finfo(np.float32).max))
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / t))
    n = len(order) if k <= 0 else min(k, len(order))
    sorted_w = w[order[:n]]
    near = 1.0
    if p < 1:
        run = np.cumsum(sorted_w)
        goal = p * run[-1]
        n = max(1, int((run - sorted_w < goal).sum()))
        near = float(np.abs(run - goal).min() / run[-1])
    kept = [i for i in order[:n] if w[i] >= m or i == order[0]]
    kept = np.sort(np.array([i for i in kept if w[i] > 0 and x[i] > -np.inf]))
    run = np.cumsum(w[kept])
    goal = u * run[-1] if u >= 0 else 0.0 if u < 0 else np.inf
    at = min(int((run <= goal).sum()), len(kept) - 1)
    if len(kept) > 1:
        near = min(near, float(np.abs(run[:-1] - goal).min() / run[-1]))
    with np.errstate(invalid="ignore"):
        y = 0.0 if x[kept[at]] == top else (x[kept[at]] - top) / t
    return kept[at], y - math.log(run[-1]), near


def _check(lm, logits, u, t=1.0, k=0, p=1.0, m=0.0, out=None, exact=False):
    rows = len(logits)
    dev = lambda v, d: torch.tensor(v, dtype=d, device="cuda") if isinstance(v, list) else v  # noqa: E731
    f = torch.float32
    args = dict(temperature=dev(t, f), top_k=dev(k, torch.int32), top_p=dev(p, f), min_p=dev(m, f))
    tokens, lp = lm.sample(logits, u, logprob=True, out=out, **args)
    again, lp2 = lm.sample(logits, u, logprob=True, **args)
    assert torch.equal(tokens.long(), again) and torch.equal(lp, lp2)
    x, uu = logits.double().cpu().numpy(), u.double().cpu().numpy()
    each = lambda v: np.float32(v if isinstance(v, list) else [v] * rows).astype(np.float64)  # noqa: E731
    t, p, m, k = each(t), each(p), each(m), k if isinstance(k, list) else [k] * rows
    for i in range(rows):
        token, logprob, near = oracle_row(x[i], uu[i], t[i], k[i], p[i], m[i])
        assert exact or near > 1e-12, "the inputs of a test have to be off the borders"
        assert int(tokens[i]) == token, (i, int(tokens[i]), token, near)
        assert abs(float(lp[i]) - logprob) <= 2.0 ** -24 * abs(logprob) + 3.5e-7, i
    return tokens, lp


def _logits(rows, vocab, dtype, seed, spread=2.5, ld=None, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or vocab
    buf = torch.full((rows * ld + offset + 8,), float("inf"), device="cuda", dtype=dtype)
    view = buf[offset:offset + rows * ld].view(rows, ld)[:, :vocab]
    view.copy_(torch.randn(rows, vocab, device="cuda", generator=g) * spread)
    return view, torch.rand(rows, device="cuda", generator=g)


SETTINGS = [dict(), dict(t=0.7), dict(k=5), dict(k=50, p=0.9), dict(p=0.8), dict(p=0.999), dict(m=0.05), dict(k=100, p=0.95, m=0.01, t=1.3), dict(t=0.0), dict(k=1), dict(p=1e-6),
            dict(k=700), dict(k=700, p=0.97), dict(t=30.0, p=0.6), dict(t=30.0, k=900)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,ld,offset", [(1, 1, 1, 0), (3, 2, 2, 0), (40, 100, 104, 0), (7, 1009, 1011, 1), (5, 4096, 4096, 0), (1, 50001, 50001, 0), (700, 300, 300, 0),
                                                  (3, 33000, 33008, 8)])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_sample(lm, dtype, rows, vocab, ld, offset, setting):
    x, u = _logits(rows, vocab, dtype, 1, 2.5, ld, offset)
    _check(lm, x, u, **SETTINGS[setting], out=torch.empty(rows, dtype=torch.int32, device="cuda") if setting % 2 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("setting", [0, 3, 4, 5, 11, 12, 13])
@pytest.mark.parametrize("spread", [0.0, 1e-6, 0.01, 1.0, 8.0, 1e4])
def test_spreads(lm, dtype, setting, spread):
    """From rows of one value, where borders fall on steps and all sums are exact, to rows with one likely token."""
    x, u = _logits(6, 9001, dtype, 2, spread)
    _check(lm, x, u, **SETTINGS[setting], exact=spread == 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_large_vocabularies(lm, dtype):
    x, u = _logits(2, 300007, dtype, 3, 1.0)
    for s in (dict(), dict(p=0.9), dict(k=2000), dict(k=50, p=0.9)):
        _check(lm, x, u, **s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("kind", ["flat", "peaked", "part_light", "part_light_peaked", "part_heavy", "equal", "masked", "lowest"])
def test_top_p_over_long_rows(lm, dtype, kind):
    """Where a part of the row (every eighth warp's vectors) says how far down top-p reaches: rows that it tells well, and rows whose part is unlike the rest."""
    x, u = _logits(5, 70001, dtype, 5, 0.0 if kind == "equal" else 6.0 if "peaked" in kind else 2.0, 70008)
    part = torch.arange(70001, device="cuda") // (32 * 16 // x.element_size()) % 8 == 0
    if "part" in kind:
        x[:, part if "light" in kind else ~part] -= 30.0
    if kind in ("masked", "lowest"):
        x[:, torch.rand(70001, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)) < 0.4] = -math.inf if kind == "masked" else torch.finfo(dtype).min
    for s in (dict(p=0.3), dict(p=0.9), dict(p=0.999), dict(p=0.9, m=0.03), dict(p=0.97, m=1e-4, t=1.5), dict(p=[0.2, 0.5, 0.8, 0.99, 1.0], t=[0.3, 0.7, 1.0, 2.0, 5.0])):
        _check(lm, x, u, **s, exact=kind == "equal")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_top_p_of_many_flat_rows(lm, dtype):
    """With tokens this light the row's weight in fp32 leaves some rows open."""
    x, u = _logits(200, 33001, dtype, 7, 1.5)
    _check(lm, x, u, p=0.9)


@pytest.mark.gpu
def test_rows_that_no_shared_memory_holds(lm):
    """2^21 logits in fp32 are read from device memory again for each pass."""
    x, u = _logits(1, (1 << 21) + 5, torch.float32, 3, 1.0)
    for s in (dict(), dict(k=3000), dict(p=0.9)):
        _check(lm, x, u, **s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [37, 5000])
def test_a_row_has_its_own_numbers(lm, dtype, vocab):
    n = 24
    x, u = _logits(n, vocab, dtype, 4)
    pick = lambda values: [values[i % len(values)] for i in range(n)]  # noqa: E731
    _check(lm, x, u, t=pick([0.5, 1.0, 0.0, 2.0, math.nan, -1.0, 0.25]), k=pick([0, 3, 20, 1, -5, 10 ** 9]), p=pick([1.0, 0.9, 0.5, 2.0]), m=pick([0.0, 0.1, 0.0, -1.0, 1.0, 1.5]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab", [50, 3001, 70001])
def test_equal_logits_go_by_their_numbers(lm, dtype, vocab):
    """Few different values: whole classes of thousands of tokens at the limit."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randint(-2, 3, (6, vocab), device="cuda", generator=g).to(dtype) * 0.5
    u = torch.rand(6, device="cuda", generator=g)
    for s in (dict(k=7), dict(k=vocab // 3), dict(p=0.3), dict(p=0.7), dict(k=vocab // 2, p=0.5), dict(m=0.4), dict(t=0.1, p=0.99)):
        _check(lm, x, u, **s, exact=True)  # a few distinct weights: sums on both sides are within 1e-13, and so are steps of at least 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_masks(lm, dtype):
    """Masked with -inf, NaN, the type's lowest value; rows of nothing, of one token, of +inf, of lowest values only, of both zeros."""
    x, u = _logits(12, 4000, dtype, 6)
    low = torch.finfo(dtype).min
    x[0, 1::2] = -math.inf
    x[1, ::3] = math.nan
    x[2, 5:] = low
    x[3] = -math.inf
    x[4] = math.nan
    x[5] = -math.inf
    x[5, 3777] = -1e30
    x[6, [5, 77, 3000]] = math.inf
    x[7] = low
    x[8] = 0.0
    x[8, ::2] = -0.0
    x[9, :3998] = -math.inf
    x[10] = math.inf
    x[11, 100:] = -math.inf
    for s in (dict(), dict(k=40), dict(p=0.9), dict(k=3, p=0.7), dict(m=0.1), dict(t=0.0), dict(k=600, p=0.99), dict(t=1e-30), dict(t=3e38)):
        tokens, _ = _check(lm, x, u, **s, exact=True)
        assert int(tokens[3]) == int(tokens[4]) == -1 and int(tokens[5]) == 3777


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_ends_of_u(lm, dtype):
    x, _ = _logits(6, 1000, dtype, 7)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -3.0, math.nan], device="cuda")
    for s in (dict(), dict(k=9), dict(p=0.5), dict(m=0.3)):
        _check(lm, x, u, **s, exact=True)


@pytest.mark.gpu
def test_extreme_logits(lm):
    """Differences that fp32 has not, temperatures as small and as large as it has them, one temperature per row."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(8, 3000, device="cuda", generator=g)
    x *= torch.tensor([1e-44, 1e-38, 1e-10, 1.0, 1e4, 1e20, 1e38, 3e38], device="cuda")[:, None] / 5
    x = x.clamp(-3.4e38, 3.4e38)
    u = torch.rand(8, device="cuda", generator=g)
    for t in ([1e-44, 1e-38, 1e-10, 1.0, 1e4, 1e20, 1e38, 3e38], [1e-45] * 8, [3.4e38] * 8, [math.inf] * 8, [1e-3] * 8):
        for s in (dict(), dict(k=30), dict(p=0.8), dict(k=1000, p=0.9)):
            _check(lm, x, u, t=t, **s, exact=True)


@pytest.mark.gpu
def test_frequencies(lm):
    """Each of 20 tokens comes as often as its probability says: 6 standard deviations of 200000 draws, which 20 tokens leave once in 2e7 runs."""
    n = 200000
    g = torch.Generator(device="cuda").manual_seed(9)
    row = torch.randn(20, device="cuda", generator=g) * 1.5
    u = torch.rand(n, device="cuda", generator=g)
    tokens = lm.sample(row.expand(n, 20).contiguous(), u, temperature=0.8)
    p = torch.softmax(row.double() / float(np.float32(0.8)), 0).cpu()
    count = torch.bincount(tokens, minlength=20).double().cpu()
    assert bool(((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 1).all())


@pytest.mark.gpu
def test_captured_and_on_another_stream(lm):
    x, u = _logits(30, 20000, torch.bfloat16, 10)
    want = lm.sample(x, u, top_p=0.9, logprob=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = lm.sample(x, u, top_p=0.9, logprob=True)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = lm.sample(x, u, top_p=0.9, logprob=True)
    third[0].zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert lm.sample(x[:0], u[:0]).shape == (0,)


@pytest.mark.gpu
def test_refusals(lm):
    from tbb_test_b200._capi import B2Error
    x, u = _logits(4, 64, torch.float32, 11)
    f = torch.ones(4, device="cuda")
    before = x.clone()
    for call in (lambda: lm.sample(x[0], u), lambda: lm.sample(x.half(), u), lambda: lm.sample(x, u[:3]), lambda: lm.sample(x, u.double()), lambda: lm.sample(x, 0.5),
                 lambda: lm.sample(x, u.cpu()), lambda: lm.sample(x, u, temperature=f[:2]), lambda: lm.sample(x, u, top_k=f), lambda: lm.sample(x, u, top_p=f.double()),
                 lambda: lm.sample(x, u, out=f), lambda: lm.sample(x, u, min_p=torch.ones(8, device="cuda")[::2])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: lm.sample(x, u, temperature=math.nan), lambda: lm.sample(x, u, top_p=math.nan), lambda: lm.sample(x, u, out=x.view(-1)[:8].view(torch.int64))):
        with pytest.raises(B2Error):
            call()
    assert torch.equal(x, before)
    out = torch.zeros(4, dtype=torch.int64, device="cuda")
    version = out._version
    assert lm.sample(x, u, out=out) is out and out._version > version


def test_c_entry_refuses_before_any_device_work(native):
    from tbb_test_b200 import _capi as K
    lib = K.lib()
    p = ct.c_void_p
    o = K.SampleOptions()
    assert lib.b2_sample_options_default(ct.byref(o)) == K.OK and o.temperature == 1.0 and o.top_k == 0 and o.top_p == 1.0 and o.min_p == 0.0 and not o.row_top_k
    assert lib.b2_sample_options_default(None) == K.ERR_INVALID

    def options(**kw):
        y = K.SampleOptions()
        lib.b2_sample_options_default(ct.byref(y))
        for k, v in kw.items():
            setattr(y, k, v)
        return ct.byref(y)

    good = dict(rows=2, vocab=8, dtype=0, x=p(256), ld=8, u=p(1024), o=options(), tokens=p(2048), size=8, lp=p(4096), ws=p(1 << 20), ws_bytes=1 << 20, stream=None)
    for kw in (dict(dtype=2), dict(rows=(1 << 24) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(size=2), dict(o=None), dict(x=None), dict(u=None), dict(tokens=None), dict(ld=7),
               dict(ws=None), dict(ws=p(64)), dict(ws_bytes=64), dict(x=p(2)), dict(u=p(2)), dict(tokens=p(4)), dict(lp=p(2)), dict(o=options(temperature=math.nan)), dict(o=options(row_top_k=2)), dict(o=options(row_top_p=2))):
        assert lib.b2_sample(*{**good, **kw}.values()) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
    need = ct.c_size_t()
    assert lib.b2_sample_workspace(2, 8, ct.byref(need)) == K.OK and need.value > 0
    assert lib.b2_sample_workspace(2, 8, None) == lib.b2_sample_workspace(2, 0, ct.byref(need)) == K.ERR_INVALID


def _check_both(lm, logits, u, **settings):
    """_check, and the same tokens by the calls without log probabilities, which go another way for rows without a limit."""
    tokens, _ = _check(lm, logits, u, **settings)
    dev = lambda v, d: torch.tensor(v, dtype=d, device="cuda") if isinstance(v, list) else v  # noqa: E731
    f = torch.float32
    again = lm.sample(logits, u, dev(settings.get("t", 1.0), f), dev(settings.get("k", 0), torch.int32), dev(settings.get("p", 1.0), f), dev(settings.get("m", 0.0), f))
    assert torch.equal(again, tokens)
    return tokens


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,ld,offset", [(300, 300, 0), (9001, 9003, 1), (70001, 70002, 3)])
def test_logits_a_few_steps_of_fp32_below_the_largest_at_a_tiny_temperature(lm, vocab, ld, offset):
    """Differences of 1 to 24 steps of fp32 with temperatures of a 1400th to a 30th of a step: most weights are below the smallest number of any type."""
    g = torch.Generator(device="cuda").manual_seed(12)
    tops, shares = [1.0, 12.0, 100.0, 1000.0, -1.0, -700.0], [1400.0, 700.0, 350.0, 100.0, 30.0, 1000.0]
    step = [2.0 ** (math.frexp(abs(v) * (1 - 2.0 ** -30))[1] - 24) for v in tops]  # of the numbers next to it that are smaller in size: finer at powers of two
    x, u = _logits(6, vocab, torch.float32, 12, 0.0, ld, offset)
    below = torch.randint(1, 25, (6, vocab), device="cuda", generator=g).double() * 2  # even: numbers larger in size than a power of two lie twice as far apart
    exact = torch.tensor(tops, device="cuda", dtype=torch.float64)[:, None] - below * torch.tensor(step, device="cuda", dtype=torch.float64)[:, None]
    assert torch.equal(exact.float().double(), exact)
    x.copy_(exact)
    x[:, torch.randint(0, vocab, (3,), device="cuda", generator=g)] = torch.tensor(tops, device="cuda")[:, None]
    for turn in range(6):
        t = [step[i] / shares[(i + turn) % 6] for i in range(6)]
        for s in (dict(), dict(k=2), dict(k=600), dict(p=0.9), dict(k=700, p=0.97), dict(m=1e-30)):
            tokens = _check_both(lm, x, u, t=t, **s, exact=True)
            assert bool(((tokens >= 0) & (tokens < vocab)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab,ld,offset", [(40, 41, 1), (3000, 3007, 3), (70001, 70003, 5)])
def test_tiny_numbers_never_take_a_masked_token(lm, dtype, vocab, ld, offset):
    """u down to fp32's smallest number, with masks and unaligned beginnings ahead of the first token that may be taken; rows with a limit beside ones without."""
    x, _ = _logits(8, vocab, dtype, 13, 2.5, ld, offset)
    x[0, 0] = x[1, :17] = x[2, :vocab - 3] = -math.inf
    x[3, :9] = math.nan
    x[4, :20] = torch.finfo(dtype).min
    x[5, :30] = -90.0  # weighs something, but less than fp32 weights tell
    x[6, 0] = x[0].max() - 79.0
    for value in (0.0, 1e-45, 1e-40, 1e-38, 1e-36, 2.3e-35, 1e-34, 1e-32, 1e-30, 1e-26, 1e-22, 1e-17, 2.0 ** -24):
        u = torch.full((8,), value, device="cuda")
        for s in (dict(), dict(t=0.5), dict(k=[0] * 7 + [3]), dict(p=[1.0] * 7 + [0.9], m=[0.0, 1e-20] * 4)):
            _check_both(lm, x, u, **s, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab,ld,offset", [(9001, 9003, 1), (40000, 40000, 0)])
@pytest.mark.parametrize("k", [5, 50, 511, 700, 3000])
def test_top_k_among_tokens_of_hardly_any_weight(lm, dtype, vocab, ld, offset, k):
    """Temperatures at which the k-th token weighs e^-40 to e^-690 of the first one: with u = 0 the token is the first kept one by number, whatever it weighs. Other rows have fewer
    tokens than k that are not masked, or thousands of equal ones at the limit."""
    x, _ = _logits(6, vocab, dtype, 14, 0.5, ld, offset)
    x[4, k // 2:] = -math.inf
    x[5].copy_((x[5].float() * 8).round() / 8)
    x[:, vocab // 2] = x.nan_to_num(neginf=-9.0).amax(1) + torch.tensor([0.0, 0.5, 1.0, 1.5, 0.5, 1.0], device="cuda").to(dtype)
    x[4, 0] = x[4, vocab // 2] - 3.0
    for value in (0.0, -1.0, 0.3):
        u = torch.full((6,), value, device="cuda")
        for s in (dict(t=0.01), dict(t=0.005), dict(t=0.01, p=0.9), dict(t=0.01, m=1e-30), dict(t=[0.01, 0.008, 0.02, 0.01, 0.01, 0.04])):
            _check_both(lm, x, u, k=k, **s, exact=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("vocab,ld,offset,spread", [(1, 1, 0, 2.5), (700, 701, 1, 2.5), (9001, 9004, 3, 0.3), (9001, 9004, 3, 9.0), (70001, 70003, 1, 2.5), (70001, 70008, 0, 9.0), (600011, 600011, 0, 0.3)])
def test_rows_without_a_limit_beside_others(lm, dtype, vocab, ld, offset, spread):
    """Settings by row, where some rows have no limit: with log probabilities and without, over tiles that are masked by -inf or by the type's lowest value, and with more tiles than
    threads."""
    n = 12
    x, u = _logits(n, vocab, dtype, 15, spread, ld, offset)
    tile = torch.arange(vocab, device="cuda") // 1024
    if vocab > 5000:
        x[1, tile % 3 != 1] = -math.inf
        x[2, tile % 2 == 0] = torch.finfo(dtype).min
        x[3, :vocab - 5] = -math.inf
        x[5, tile < tile[-1] // 2] = -30.0 - spread * 10
    pick = lambda values: [values[i % len(values)] for i in range(n)]  # noqa: E731
    k, p, m = [0] * 9 + [20, 0, 0], [1.0] * 10 + [0.9, 1.0], [0.0] * 11 + [0.05]
    _check_both(lm, x, u, t=pick([1.0, 0.5, 1.0, 2.0, 0.25]), k=k, p=p, m=m)
    _check_both(lm, x, u, t=pick([1.0, 0.0, math.nan, 1e30, 1e-30]), p=p, exact=True)
    _check_both(lm, x, u, m=m)
    many = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(16))
    _check_both(lm, x, many, k=k, p=p)


@pytest.mark.gpu
def test_log_probabilities_over_the_whole_range_of_fp32_powers(lm):
    """The bound of fp32 weights: two tokens in different tiles, the second of them as a power of two with a fraction anywhere in +-1/2, against the logarithm in 64 bits."""
    n = 1 << 14
    x = torch.full((n, 1100), -math.inf, device="cuda")
    x[:, 0] = 0.0
    x[:, 1050] = -torch.linspace(1e-4, 2.1, n, device="cuda")
    tokens, lp = lm.sample(x, torch.zeros(n, device="cuda"), logprob=True)
    want = -torch.log1p(torch.exp(x[:, 1050].double()))
    assert not tokens.any() and bool(((lp.double() - want).abs() <= 2.0 ** -24 * want.abs() + 3.5e-7).all())
