"""Root-mean-square norm, its 8-bit output and its gradients (tbb_test_b200.lm) against the formulas in 64 bits.

Tolerances, counted in u = 2^-24 (half a step of fp32, relative). A vector of at most 8 squares is summed in fp32 (8 u, terms of one sign) and
vectors in fp64; r = 1 / sqrt(mean + eps) gets half of that, half a u from the mean's conversion and one each from root and quotient: 6.5 u. n = t r one
more, y = n w one more: 8.5 u, taken as 9 u. An output's own rounding is half a step of its type (bf16 2^-8)."""
import ctypes as ct
import math

import pytest

torch = pytest.importorskip("torch")

DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24
EPS = {k: torch.finfo(v).eps / 2 for k, v in DTYPE.items()}


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _rows(n, d, dtype, seed, ld=None, offset=0, scale=1.0):
    """n x d values, as a view into a buffer with other rows and columns of NaN around it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or d
    buf = torch.full((n * ld + offset + 8,), float("nan"), device="cuda", dtype=DTYPE[dtype])
    view = buf[offset:offset + n * ld].view(n, ld)[:, :d]
    view.copy_(torch.randn(n, d, device="cuda", generator=g) * scale * (0.1 + torch.rand(n, 1, device="cuda", generator=g)))
    return view


def _weight(d, kind, dtype, offset=0):
    if kind is None:
        return None
    g = torch.Generator(device="cuda").manual_seed(77)
    t = DTYPE[dtype] if kind == "same" else torch.float32
    buf = torch.full((d + offset,), float("nan"), device="cuda", dtype=t)
    buf[offset:] = 1 + 0.5 * torch.randn(d, device="cuda", generator=g)
    return buf[offset:]


def _exact(t, w, eps):
    t = t.double()
    r = 1.0 / torch.sqrt(t.square().mean(1, keepdim=True) + eps)
    n = t * r
    return n if w is None else n * w.double(), n, r


# rows, width, leading dimension, offset in elements: whole 16-byte pieces, narrower vectors and single elements; a group of one thread, of a warp,
# of several warps, of a block; rows longer than registers hold
SHAPES = [(1, 1, 1, 0), (5, 8, 8, 0), (3, 3, 7, 1), (300, 16, 24, 0), (77, 203, 203, 0), (1000, 64, 64, 0), (33, 130, 134, 2), (9, 1024, 1024, 0),
          (2, 1000, 1004, 4), (4, 4096, 4104, 0), (1, 5000, 5001, 1), (3, 8192, 8192, 0), (2, 10007, 10007, 0), (2, 16384, 16384, 0), (2, 40000, 40000, 0),
          (1500, 128, 128, 0), (700, 520, 520, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,width,ld,offset", SHAPES)
@pytest.mark.parametrize("weight,residual", [("same", True), ("fp32", False), (None, True)])
def test_norm(lm, dtype, rows, width, ld, offset, weight, residual):
    x = _rows(rows, width, dtype, 1, ld, offset)
    res = _rows(rows, width, dtype, 2, ld, offset) if residual else None
    w = _weight(width, weight, dtype, offset)
    out = _rows(rows, width, dtype, 3, ld, offset)
    eps = 1e-5
    if residual:
        total = _rows(rows, width, dtype, 4, ld, offset)
        got, t = lm.norm(x, w, res, eps=eps, total=total, out=out)
        assert got is out and t is total
        assert torch.equal(t, (x.float() + res.float()).to(x.dtype))
        again, t2 = lm.norm(x.contiguous(), w, res.contiguous(), eps=eps)
        assert torch.equal(t2, t)
        assert torch.equal(lm.norm(total, w, eps=eps, out=_rows(rows, width, dtype, 3, ld, offset)), out)  # it is the norm of exactly what was written
    else:
        assert lm.norm(x, w, eps=eps, out=out) is out
        t, again = x, lm.norm(x.contiguous(), w, eps=eps)
    want = _exact(t, w, eps)[0]
    tolerance = want.abs() * (9 * U + EPS[dtype])
    assert bool(((out.double() - want).abs() <= tolerance).all())
    assert bool(((again.double() - want).abs() <= tolerance).all())
    if ld > width:  # what lies between and behind the rows is left as it was
        assert bool(torch.isnan(out.as_strided((rows - 1, ld - width), (ld, 1), out.storage_offset() + width)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,width,ld,offset", SHAPES)
@pytest.mark.parametrize("block,residual", [(128, True), (0, False)])
def test_e4m3(lm, dtype, rows, width, ld, offset, block, residual):
    x = _rows(rows, width, dtype, 1, ld, offset)
    x[rows // 2] = 0.0
    res = _rows(rows, width, dtype, 2, ld, offset) if residual else None
    w = _weight(width, "fp32" if residual else "same", dtype, offset)
    if residual:
        q, scales, t = lm.norm_e4m3(x, w, res, eps=1e-5, block=block)
        assert torch.equal(t, (x.float() + res.float()).to(x.dtype))
    else:
        q, scales = lm.norm_e4m3(x, w, eps=1e-5, block=block)
        t = x
    assert q.dtype == torch.float8_e4m3fn and q.shape == (rows, width) and scales.shape == (rows, -(-width // block) if block else 1)
    y = _exact(t, w, 1e-5)[0]
    step = block or width
    for i, part in enumerate(y.split(step, 1)):
        scale = (part.abs().amax(1) / 448).clamp(min=2.0 ** -126)
        assert bool(((scales[:, i].double() - scale).abs() <= 10 * U * scale).all())  # y's 9 u and the quotient's own
        v = part / scale[:, None]
        # half a step of three bits behind the leading one (2^-10 below 2^-6); v's own 9 + 10 u and the quotient's may also bring it over a power of two
        v_most = v.abs() * (1 + 20 * U)
        half = torch.exp2(torch.floor(torch.log2(v_most.clamp(min=2.0 ** -6))) - 4)
        assert bool(((q[:, i * step:i * step + part.shape[1]].double() - v).abs() <= half + 20 * U * v.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,width,ld,offset", SHAPES)
@pytest.mark.parametrize("weight,more", [("same", True), ("fp32", False), (None, True)])
def test_gradients(lm, dtype, rows, width, ld, offset, weight, more):
    """dx = r (g - n c) + dtotal: g one rounding, n 7.5 u; c = r mean(g t): products and sums of 8 in fp32 9 u of the magnitudes, r 6.5 u, its own
    conversion 1 u; the product n c, the difference, r's and dtotal's sum one each: 30 u of r (|g| + |n| mean|g n|) cover them. dw: each term 9.5 u, and any order
    of `rows` additions."""
    eps = 1e-5
    t, dy = _rows(rows, width, dtype, 1, ld, offset), _rows(rows, width, dtype, 2, ld, offset, 1e-3)
    dy[rows // 3] = 0.0
    dt = _rows(rows, width, dtype, 3, ld, offset, 1e-3) if more else None
    w = _weight(width, weight, dtype, offset)
    dx = _rows(rows, width, dtype, 4, ld, offset)
    got = lm.norm_grad(dy, t, w, dt, eps=eps, dx=dx)
    again = lm.norm_grad(dy, t, w, dt, eps=eps)
    if w is None:
        assert got is dx and torch.equal(again, dx)
    else:
        assert got[0] is dx and torch.equal(again[0], dx) and torch.equal(again[1], got[1])  # the same bits
    _, n, r = _exact(t, w, eps)
    g = dy.double() if w is None else dy.double() * w.double()
    want = r * (g - n * (g * n).mean(1, keepdim=True)) + (0.0 if dt is None else dt.double())
    size = r * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
    tolerance = 30 * U * size + (0.0 if dt is None else 2 * U * dt.double().abs()) + EPS[dtype] * want.abs() * 1.01
    assert bool(((dx.double() - want).abs() <= tolerance).all())
    if w is not None:
        dw = got[1]
        assert dw.dtype == w.dtype
        terms = dy.double() * n
        want = terms.sum(0)
        assert bool(((dw.double() - want).abs() <= (rows + 10) * U * terms.abs().sum(0) + torch.finfo(dw.dtype).eps / 2 * want.abs() * 1.01).all())


@pytest.mark.gpu
def test_gradients_against_differences(lm):
    """<dy, y(t + h d) - y(t - h d)> / 2h in 64 bits of the formula, whose third derivatives at h = 1e-5 are far below the tolerance."""
    t, dy, w = _rows(40, 72, "fp32", 1), _rows(40, 72, "fp32", 2), _weight(72, "fp32", "fp32")
    dx, dw = lm.norm_grad(dy, t, w, eps=1e-3)
    g = torch.Generator(device="cuda").manual_seed(5)
    h = 1e-5
    for _ in range(5):
        d, e = (torch.randn(*s, device="cuda", generator=g, dtype=torch.float64) for s in ((40, 72), (72,)))
        f = lambda k: (dy.double() * _exact(t.double() + k * h * d, w.double() + k * h * e, 1e-3)[0]).sum()  # noqa: E731
        want = float(f(1) - f(-1)) / (2 * h)
        got = float((dx.double() * d).sum() + (dw.double() * e).sum())
        size = float((dx.double() * d).abs().sum() + (dw.double() * e).abs().sum())
        assert abs(got - want) <= 60 * U * size * 40 + 1e-7 * size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [24, 203, 1024, 40000])
def test_the_whole_range(lm, dtype, width):
    """Squares that fp32 has not: rows of 1e-38 to 1e38, one row of zeros, and eps far below or zero. Results below 2^-126 are off by up to half of
    fp32's smallest step (2^-150) or bf16's (2^-134)."""
    scales = torch.tensor([1e-38, 1e-30, 1e-20, 1e-3, 1.0, 1e10, 1e20, 1e30, 3e37], device="cuda")[:, None]
    t = _rows(9, width, dtype, 1).contiguous()
    t = (t.float().clamp(-3, 3) * scales).to(DTYPE[dtype])
    least = 2.0 ** -134 if dtype == "bf16" else 2.0 ** -150
    for eps in (0.0, 1e-35, 1e-6):
        y = lm.norm(t, eps=float(eps))
        want = _exact(t, None, float(torch.tensor(eps, dtype=torch.float32)))[0]
        assert bool(((y.double() - want).abs() <= want.abs() * (9 * U + EPS[dtype]) + least).all())
        dy = _rows(9, width, dtype, 2)
        dx = lm.norm_grad(dy, t, eps=float(eps))
        _, n, r = _exact(t, None, float(torch.tensor(eps, dtype=torch.float32)))
        g = dy.double()
        want = r * (g - n * (g * n).mean(1, keepdim=True))
        size = r * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
        most = torch.finfo(DTYPE[dtype]).max
        fits = size < 0.5 * most
        assert bool(((dx.double() - want).abs() <= 30 * U * size + EPS[dtype] * want.abs() * 1.01 + least)[fits].all()) and bool(fits[2:].all())
    z = torch.zeros(2, width, device="cuda", dtype=DTYPE[dtype])
    assert not lm.norm(z, eps=1e-6).any()
    q, s = lm.norm_e4m3(z, eps=1e-6)
    assert not q.float().any() and bool((s == 2.0 ** -126).all())


@pytest.mark.gpu
def test_small_gradients_keep_their_bits(lm):
    """Products of gradient and input below fp32's smallest number: their mean still counts."""
    t, dy = _rows(7, 96, "fp32", 1) * 1e-10, _rows(7, 96, "fp32", 2) * 1e-33
    dx = lm.norm_grad(dy, t, eps=1e-24)
    _, n, r = _exact(t, None, float(torch.tensor(1e-24)))
    g = dy.double()
    want = r * (g - n * (g * n).mean(1, keepdim=True))
    size = r * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
    assert bool(((dx.double() - want).abs() <= 30 * U * size + 1e9 * 2.0 ** -149).all())


@pytest.mark.gpu
def test_nan_and_inf_stay_in_their_rows(lm):
    t = _rows(6, 200, "fp32", 1).contiguous()
    clean = lm.norm(t)
    bad = t.clone()
    bad[1, 3], bad[4, 7] = float("nan"), float("inf")
    y = lm.norm(bad)
    assert torch.equal(y[[0, 2, 3, 5]], clean[[0, 2, 3, 5]]) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[4, 7])) and not y[4, :7].any()
    dy = _rows(6, 200, "fp32", 2)
    assert torch.equal(lm.norm_grad(dy, bad)[[0, 2, 3, 5]], lm.norm_grad(dy, t)[[0, 2, 3, 5]])


@pytest.mark.gpu
def test_no_rows(lm):
    x, w = torch.empty(0, 40, device="cuda"), torch.ones(40, device="cuda")
    assert lm.norm(x, w).shape == (0, 40)
    q, s = lm.norm_e4m3(x, w)
    assert q.shape == (0, 40) and s.shape == (0, 1)
    dx, dw = lm.norm_grad(x, x, w)
    assert dx.shape == (0, 40) and not dw.any()


@pytest.mark.gpu
def test_captured_and_on_another_stream(lm):
    x, res, w = _rows(300, 512, "bf16", 1), _rows(300, 512, "bf16", 2), _weight(512, "fp32", "bf16")
    dy = _rows(300, 512, "bf16", 3)
    y, t = lm.norm(x, w, res)
    dx, dw = lm.norm_grad(dy, t, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2, t2 = lm.norm(x, w, res)
        dx2, dw2 = lm.norm_grad(dy, t2, w)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y3, t3 = lm.norm(x, w, res)
        dx3, dw3 = lm.norm_grad(dy, t3, w)
    for v in (y3, dx3, dw3):
        v.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for want, *got in ((y, y2, y3), (t, t2, t3), (dx, dx2, dx3), (dw, dw2, dw3)):
        assert all(torch.equal(want, v) for v in got)


@pytest.mark.gpu
def test_wrapper_refuses(lm):
    x, w = torch.zeros(4, 16, device="cuda"), torch.zeros(16, device="cuda")
    h = x.bfloat16()
    for call in (lambda: lm.norm(x.half()), lambda: lm.norm(x[0]), lambda: lm.norm(x, w[:8]), lambda: lm.norm(x, w.bfloat16()), lambda: lm.norm(x, w.cpu()),
                 lambda: lm.norm(x, w, x[:2]), lambda: lm.norm(x, w, h), lambda: lm.norm(x, total=x), lambda: lm.norm(x.mT), lambda: lm.norm(x.cpu()),
                 lambda: lm.norm_e4m3(x, block=64), lambda: lm.norm_grad(x, h), lambda: lm.norm_grad(x, x, dtotal=x[:1]), lambda: lm.norm(x, out=h),
                 lambda: lm.norm(x, torch.zeros(32, device="cuda")[::2])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_overlaps_are_refused(lm):
    from tbb_test_b200._capi import B2Error
    x, r, w, o = (torch.ones(4, 16, device="cuda") for _ in range(4))
    for call in (lambda: lm.norm(x, out=x), lambda: lm.norm(x, w[0], r, total=r), lambda: lm.norm(x, w[0], r, total=o, out=o), lambda: lm.norm(x, w[0], out=w),
                 lambda: lm.norm_grad(x, r, dx=x), lambda: lm.norm_grad(x, r, dx=r), lambda: lm.norm_grad(x, r, w[0], o, dx=o), lambda: lm.norm_grad(x, r, w[0], dx=w)):
        with pytest.raises(B2Error, match="overlap"):
            call()
    torch.cuda.synchronize()
    assert all(bool((v == 1).all()) for v in (x, r, w, o))


def test_c_entries_refuse_before_any_device_work(native):
    from tbb_test_b200 import _capi as K
    lib = K.lib()
    p = ct.c_void_p
    good = dict(rows=2, width=8, dtype=0, x=p(256), ldx=8, r=p(512), ldr=8, w=p(1024), wt=0, eps=1e-6, t=p(2048), ldt=8, ot=0, o=p(4096), ldo=8, s=p(8192), lds=1,
                block=0, stream=None)
    for kw in (dict(dtype=2), dict(dtype=1), dict(wt=1), dict(rows=1 << 31), dict(width=0), dict(width=(1 << 20) + 1), dict(eps=-1.0), dict(eps=math.nan),
               dict(eps=math.inf), dict(ot=1), dict(ot=3), dict(ot=2, block=64), dict(ot=2, s=None), dict(ot=2, s=p(3)), dict(ot=2, lds=0), dict(r=None), dict(x=None),
               dict(o=None), dict(ldx=7), dict(ldr=7), dict(ldt=7), dict(ldo=7), dict(x=p(2)), dict(t=p(2)), dict(o=p(2)), dict(w=p(2)),
               dict(ot=2, block=128, width=129, ldx=129, ldr=129, ldt=129, ldo=129)):
        assert lib.b2_norm(*{**good, **kw}.values()) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
    need = ct.c_size_t()
    assert lib.b2_norm_grad_workspace(2, 8, 0, ct.byref(need)) == K.OK and need.value > 0
    assert lib.b2_norm_grad_workspace(2, 8, 0, None) == lib.b2_norm_grad_workspace(2, 8, 5, ct.byref(need)) == K.ERR_INVALID
    good = dict(rows=2, width=8, dtype=0, dy=p(256), ldy=8, t=p(512), ldt=8, m=p(1024), ldm=8, w=p(2048), wt=0, eps=1e-6, dx=p(4096), ldx=8, dw=p(8192), ws=p(1 << 20),
                ws_bytes=1 << 30, stream=None)
    for kw in (dict(dtype=2), dict(wt=1), dict(width=0), dict(eps=-1.0), dict(w=None), dict(dy=None), dict(t=None), dict(dx=None), dict(ws=None), dict(ldy=7), dict(ldt=7),
               dict(ldm=7), dict(ldx=7), dict(dy=p(1)), dict(dw=p(2)), dict(ws=p(64)), dict(ws_bytes=100)):
        assert lib.b2_norm_grad(*{**good, **kw}.values()) == K.ERR_INVALID, kw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [v * n for n in (1, 2, 4, 8) for v in (1, 512, 513, 2048, 2049, 4095, 4097)])
def test_gradients_at_the_ends_of_their_forms(lm, dtype, width):
    """Rows of so many vectors of 1, 2, 4 or 8 elements: as many as 256 threads hold with two each or with all that they may, 1024 threads, and one more."""
    test_gradients(lm, dtype, 3, width, width, 0, "fp32", True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width", [203, 1024, 40000])
@pytest.mark.parametrize("block", [0, 128])
def test_e4m3_of_infinite_elements_and_over_the_whole_range(lm, dtype, width, block):
    """Norms of 1e-38 to 1e38 by their weights. A block with an infinite norm has an infinite scale, behind which the finite ones are 0; NaN stays where it is and scales nothing."""
    x = _rows(4, width, dtype, 1).contiguous()
    w = torch.ones(width, device="cuda")
    for factor in (1e-38, 1e-30, 1e30, 2e36):
        q, scales = lm.norm_e4m3(x, w * factor, block=block)
        y = _exact(x, w * factor, float(torch.tensor(1e-6)))[0]
        s = scales.double().repeat_interleave(block or width, 1)[:, :width]
        assert bool(torch.isfinite(scales).all())
        # three bits behind the leading one, or half of 2^-9 scales below 2^-6 of them; y's own 9 u and the scale's 10 u
        assert bool(((q.double() * s - y).abs() <= y.abs() * (2.0 ** -4 + 20 * U) + 2.0 ** -10 * s * (1 + 20 * U)).all())
    clean_q, clean_s = lm.norm_e4m3(x, w, block=block)
    bad = w.clone()
    bad[3], bad[7] = math.inf, math.nan
    q, scales = lm.norm_e4m3(x, bad, block=block)
    here = block or width
    assert bool(torch.isinf(scales[:, 0]).all()) and torch.equal(scales[:, 1:], clean_s[:, 1:]) and torch.equal(q[:, here:].float(), clean_q[:, here:].float())
    first = q[:, :min(here, width)].float()
    assert bool(torch.isnan(first[:, [3, 7]]).all()) and not first[:, :3].any() and not first[:, 8:].any()
    bad[3] = 1.0
    q, scales = lm.norm_e4m3(x, bad, block=block)
    assert bool(torch.isfinite(scales).all()) and bool(torch.isnan(q.float()[:, 7]).all()) and int(torch.isnan(q.float()).sum()) == 4
