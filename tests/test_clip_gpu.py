"""The global norm of a list of tensors and their clipping (tbb_test_b200.lm.clip) against the formulas in 64 bits.

In u = 2^-24: vectors of at most 8 squares are summed in fp32 (8 u), everything else in fp64: the norm gets half of it and its own rounding, 5 u. The
factor gets the norm's 4 u and its own rounding, the product one more: 6 u, and the output's rounding in its type."""
import ctypes as ct
import math

import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -24


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _make(sizes, seed, scale=1.0, dtypes=(torch.float32, torch.bfloat16)):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def _norm(xs):
    return math.sqrt(sum(float(x.double().square().sum()) for x in xs))


def _check(xs, before, norm, max_norm):
    want = _norm(before)
    assert abs(float(norm) - want) <= 5 * U * want
    factor = min(1.0, float(torch.tensor(max_norm)) / want) if want else 1.0
    for x, b in zip(xs, before):
        exact = b.double() * factor
        eps = torch.finfo(x.dtype).eps / 2
        assert x.shape == b.shape and bool(((x.double() - exact).abs() <= exact.abs() * (6 * U + eps)).all())


LISTS = {"one": [(1,)], "scalars": [(), (), (1, 1)], "odd": [(203,), (7, 31), (1000, 203), (3, 5, 7), (0, 4), (1,)], "many": [(1 + 37 * i % 5000,) for i in range(700)],
         "forty": [(64, 33)] * 40, "forty-one": [(17,)] * 41, "large": [(2048, 2048), (4096,), (1023, 4097)], "empty": [(0,), (3, 0)]}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)], ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.5])
def test_clip(lm, name, dtypes, share):
    xs = _make(LISTS[name], 1, dtypes=dtypes)
    before = [x.clone() for x in xs]
    limit = float(torch.tensor(_norm(xs) * share))
    outs = [torch.full_like(x, 7) for x in xs]
    n1 = lm.clip(xs, limit, out=outs)
    assert all(torch.equal(x, b) for x, b in zip(xs, before))
    _check(outs, before, n1, limit)
    n2 = lm.clip(xs, limit)
    assert torch.equal(n1, n2) and all(torch.equal(x, o) for x, o in zip(xs, outs))
    if share > 1:
        assert all(torch.equal(x, b) for x, b in zip(xs, before))
    for none in (None, math.inf):
        assert torch.equal(lm.clip(before, none), n1)
    assert n1.dtype == torch.float32 and n1.shape == () and n1.device == xs[0].device


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_alignment(lm, dtype):
    """Tensors and outputs that begin anywhere, alike or not; what lies beside them stays."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for a in range(9):
        for b in (a, 0, 1, 2, 3, 4):
            sizes = [1, 2, 3, 7, 8, 9, 33, 5000, 4096 + a]
            x, y = (torch.randn(sum(sizes) + 40, device="cuda", generator=g).to(dtype) for _ in range(2))
            x0, y0 = x.clone(), y.clone()
            xs, ys, at = [], [], 0
            for s in sizes:
                xs.append(x[at + a:at + a + s])
                ys.append(y[at + b:at + b + s])
                at += s
            norm = lm.clip(xs, 1.5, out=ys)
            _check(ys, xs, norm, 1.5)
            assert torch.equal(x, x0) and torch.equal(y[:b], y0[:b]) and torch.equal(y[b + at:], y0[b + at:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_with_gaps_and_other_orders(lm, dtype):
    g = torch.Generator(device="cuda").manual_seed(4)
    buf = torch.randn(300, 200, device="cuda", generator=g).to(dtype)
    other = torch.randn(70, 90, 11, device="cuda", generator=g).to(dtype)
    xs = [buf[:, :100], buf[7:100, 103:104], buf[:200, 120:199], other.permute(2, 0, 1), other.new_ones(5, 1)[:, :1]]
    whole, whole2, before = buf.clone(), other.clone(), [x.clone() for x in xs]
    outs = [torch.empty(300, 120, device="cuda", dtype=dtype)[:, :100], torch.empty(93, 1, device="cuda", dtype=dtype), torch.empty(200, 79, device="cuda", dtype=dtype),
            torch.empty_like(xs[3]), torch.empty(5, 1, device="cuda", dtype=dtype)]
    norm = lm.clip(xs, 2.0, out=outs)
    assert torch.equal(buf, whole) and torch.equal(other, whole2)
    _check(outs, before, norm, 2.0)
    assert torch.equal(lm.clip(xs, 2.0), norm)
    assert all(torch.equal(x, o) for x, o in zip(xs, outs))
    rest = torch.ones_like(buf, dtype=torch.bool)
    rest[:, :100] = rest[7:100, 103:104] = rest[:200, 120:199] = False
    assert torch.equal(buf[rest], whole[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-20, 1e18, 1e30])
def test_the_whole_range(lm, scale):
    xs = _make([(1000, 30), (999,)], 5)
    xs = [(x.double().clamp(-3, 3) * scale).to(x.dtype) for x in xs]
    before = [x.clone() for x in xs]
    limit = float(torch.tensor(_norm(xs) * 0.25))
    norm = lm.clip(xs, limit)
    want = _norm(before)
    assert abs(float(norm) - want) <= 5 * U * want
    for x, b in zip(xs, before):
        least = 2.0 ** -150 if x.dtype == torch.float32 else 2.0 ** -134  # half of the type's smallest step
        exact = b.double() * (limit / want)
        assert bool(((x.double() - exact).abs() <= exact.abs() * (6 * U + torch.finfo(x.dtype).eps / 2) + least).all())


@pytest.mark.gpu
@pytest.mark.parametrize("what", [math.inf, math.nan])
def test_what_is_not_finite_changes_nothing(lm, what):
    xs = _make([(500,), (600,)], 6)
    xs[1][77] = what
    before = [x.clone() for x in xs]
    outs = [torch.zeros_like(x) for x in xs]
    n = [lm.clip(xs, 0.5), lm.clip(xs, 0.5, out=outs)]
    for v in n:
        assert math.isinf(float(v)) if math.isinf(what) else math.isnan(float(v))
    for x, o, b in zip(xs, outs, before):
        assert torch.equal(x.nan_to_num(5.0), b.nan_to_num(5.0)) and torch.equal(o.nan_to_num(5.0), b.nan_to_num(5.0))


@pytest.mark.gpu
def test_zeros(lm):
    xs = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda")]
    for limit in (0.0, 1.0):
        assert float(lm.clip(xs, limit)) == 0.0 and not any(x.any() for x in xs)


@pytest.mark.gpu
def test_captured_and_on_another_stream(lm):
    xs = _make([(1 + 991 * i % 70001,) for i in range(60)], 7)
    outs = [torch.empty_like(x) for x in xs]
    norm = lm.clip(xs, 1.0, out=outs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [x.clone() for x in xs]
        n2 = lm.clip(again, 1.0)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    third = [x.clone() for x in xs]
    with torch.cuda.graph(graph):
        n3 = lm.clip(third, 1.0)
    for _ in range(2):
        for x, y in zip(xs, third):
            y.copy_(x)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, n2) and torch.equal(norm, n3)
    assert all(torch.equal(o, a) and torch.equal(o, b) for o, a, b in zip(outs, again, third))


@pytest.mark.gpu
def test_autograds_count_of_changes(lm):
    x = torch.randn(30, device="cuda", requires_grad=True)
    y = (x * x).sum()
    lm.clip([x.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    z = (x * x).sum()
    lm.clip([x.detach()], None)
    z.backward()
    with torch.inference_mode():
        assert not lm.clip([x.detach().clone()], 1.0).requires_grad


@pytest.mark.gpu
def test_refusals(lm):
    from tbb_test_b200._capi import B2Error
    x = torch.ones(8, 16, device="cuda")
    for call in (lambda: lm.clip([], 1.0), lambda: lm.clip([x.half()], 1.0), lambda: lm.clip([x.cpu()], 1.0), lambda: lm.clip([x, x.cpu()], 1.0), lambda: lm.clip([x], -1.0),
                 lambda: lm.clip([x], math.nan), lambda: lm.clip([x], 1.0, out=[]), lambda: lm.clip([x], 1.0, out=[x[:4]]), lambda: lm.clip([x], 1.0, out=[x.bfloat16()]),
                 lambda: lm.clip([x], None, out=[x.clone()]), lambda: lm.clip([x[:, ::2]], 1.0), lambda: lm.clip([x[:1].expand(8, 16)], 1.0),
                 lambda: lm.clip([x.mT], 1.0, out=[x.mT.contiguous()]), lambda: lm.clip([3.0], 1.0)):
        with pytest.raises(ValueError):
            call()
    y = torch.ones(8, 16, device="cuda")
    for call in (lambda: lm.clip([x, x], 0.1), lambda: lm.clip([x, x[3]], 0.1), lambda: lm.clip([x, y], 0.1, out=[y, x]), lambda: lm.clip([x[:4]], 0.1, out=[x[2:6]]),
                 lambda: lm.clip([x[:, :8], x[:, 7:12]], 0.1)):
        with pytest.raises(B2Error, match="overlap"):
            call()
    torch.cuda.synchronize()
    assert bool((x == 1).all()) and bool((y == 1).all())
    assert abs(float(lm.clip([x, x], None)) - 16.0) <= 16 * 5 * U  # read only: twice is allowed


def test_c_entry_refuses_before_any_device_work(native):
    from tbb_test_b200 import _capi as K
    lib = K.lib()
    p = ct.c_void_p
    ptr = lambda *v: (ct.c_void_p * 2)(*v)  # noqa: E731
    num = lambda *v: (ct.c_size_t * 2)(*v)  # noqa: E731
    good = dict(count=2, x=ptr(256, 4096), out=ptr(256, 4096), elements=num(16, 16), dtypes=(ct.c_int * 2)(0, 0), widths=num(8, 8), ld_x=num(8, 8), ld_out=num(8, 8),
                max_norm=1.0, norm=p(1 << 16), ws=p(1 << 20), ws_bytes=1 << 20, stream=None)
    for kw in (dict(count=(1 << 20) + 1), dict(x=None), dict(elements=None), dict(dtypes=None), dict(ld_x=None), dict(ld_out=None), dict(max_norm=-1.0), dict(max_norm=math.nan),
               dict(norm=None), dict(norm=p(2)), dict(ws=None), dict(ws=p(64)), dict(ws_bytes=16), dict(dtypes=(ct.c_int * 2)(0, 2)), dict(x=ptr(256, None)),
               dict(out=ptr(256, None)), dict(x=ptr(256, 4098)), dict(out=ptr(256, 4098)), dict(ld_x=num(8, 7)), dict(ld_out=num(8, 7)), dict(widths=num(8, 5)),
               dict(widths=num(8, 0)), dict(elements=num(16, (1 << 42) + 1)), dict(elements=num(1 << 41, (1 << 41) + 8)), dict(max_norm=math.inf)):
        assert lib.b2_clip(*{**good, **kw}.values()) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
    need = ct.c_size_t()
    assert lib.b2_clip_workspace(700, ct.byref(need)) == K.OK and need.value > 0
    assert lib.b2_clip_workspace(1, None) == lib.b2_clip_workspace((1 << 20) + 1, ct.byref(need)) == K.ERR_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_norm_beyond_fp32_is_infinite_and_changes_nothing(lm, dtype):
    """Two elements of 3e38: each is finite, their norm is not in fp32. One of 3e38 beside it is clipped as ever."""
    xs = [torch.tensor([3e38, 1.0], device="cuda").to(dtype), torch.tensor([-2.0, 3e38, 5.0], device="cuda").to(dtype)]
    before, outs = [x.clone() for x in xs], [torch.zeros_like(x) for x in xs]
    for norm in (lm.clip(xs, 1.0), lm.clip(xs, 1.0, out=outs), lm.clip(xs, None)):
        assert math.isinf(float(norm))
    assert all(torch.equal(x, b) and torch.equal(o, b) for x, o, b in zip(xs, outs, before))
    _check(xs[:1], before[:1], lm.clip(xs[:1], 1e38), 1e38)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("scale,limit", [(1e30, 1e-12), (1e30, 1e-16), (1e36, 1e-6), (3e30, 1e-35), (1e-3, 1e-44), (1e20, 1e-17), (1.0, 1e-38)])
def test_limits_far_below_the_norm(lm, dtype, scale, limit):
    """Factors that fp32 has not, or not with all of its bits, among dense tensors and matrices with gaps, in place and not. Results below the type's normal numbers are off by
    up to half of its smallest step; through fp32, bf16 by half of fp32's more."""
    g = torch.Generator(device="cuda").manual_seed(8)
    buf = (torch.randn(70, 50, device="cuda", generator=g).clamp(-3, 3) * scale).to(dtype)
    xs = [buf[:, :33], (torch.randn(5003, device="cuda", generator=g).clamp(-3, 3) * scale).to(dtype)[1:], buf[3:4, 40:41]]
    before, rest = [x.clone() for x in xs], buf[:, 41:].clone()
    limit = float(torch.tensor(limit))
    outs = [torch.full_like(x, 7) for x in xs]
    norm = lm.clip(xs, limit, out=outs)
    assert torch.equal(lm.clip(xs, limit), norm) and all(torch.equal(x, o) for x, o in zip(xs, outs)) and torch.equal(buf[:, 41:], rest)
    want = _norm(before)
    assert abs(float(norm) - want) <= 5 * U * want
    least = 2.0 ** -150 if dtype == torch.float32 else 2.0 ** -134 + 2.0 ** -150
    for o, b in zip(outs, before):
        exact = b.double() * (limit / want)
        assert bool(((o.double() - exact).abs() <= exact.abs() * (6 * U + torch.finfo(dtype).eps / 2) + least).all())


@pytest.mark.gpu
def test_limits_beyond_fp32(lm):
    """Finite in a Python number: outputs are written, and nothing is over such a limit."""
    x, out = torch.full((9,), 1e38, device="cuda"), torch.zeros(9, device="cuda")
    assert abs(float(lm.clip([x], 1e39, out=[out])) - 3e38) <= 3e38 * 5 * U and torch.equal(out, x)
    assert float(lm.clip([x], 3.5e38)) < math.inf and bool((x == 1e38).all())
