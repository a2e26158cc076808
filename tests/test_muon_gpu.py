"""The orthogonalised update (tbb_test_b200.lm.muon) against its formula in 64 bits.

Tolerances, in Frobenius norm, from the arithmetic. The step f(x) = (A I + B a + C a a) x maps singular values by
p(s) = A s + B s^3 + C s^5, so an error before a step leaves it at most L = 3.9 times as large (the largest |p'| for
s in [0, 1.21], where all singular values stay). A step's own products, each at 2^-20 (22-bit operands, fp32 sums), add
(A + 3 |B| + 5 C) 2^-20 |x|. The start has an error of 2^-20. Momentum is one product and one sum in fp32."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

A, B, C = 3.4445, -4.7750, 2.0315
L, UNIT = 3.9, 2.0 ** -20
OWN = (A + 3 * abs(B) + 5 * C) * UNIT


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _exact(w, m, g, lr, mu, nesterov, decay, scale, eps, steps=5):
    """New weights and momentum in 64 bits, and the bound on the update's error."""
    m = mu * m + g
    u = g + mu * m if nesterov else m
    x = u / (torch.linalg.norm(u) + eps)
    off = UNIT * float(torch.linalg.norm(x))
    for _ in range(steps):
        off = L * off + OWN * float(torch.linalg.norm(x))
        x = A * x + B * (x @ x.T @ x) + C * (x @ x.T @ x @ x.T @ x)
    return w * (1 - lr * decay) - lr * scale * x, m, abs(lr * scale) * off


def _check(before, after, o):
    (w, m, g), (w2, m2, copy) = before, after
    f = {k: float(np.float32(o[k])) for k in ("lr", "momentum", "weight_decay", "scale", "eps")}
    for i in range(len(w)):
        want, mom, off = _exact(w[i].double(), m[i].double(), g[i].double(), f["lr"], f["momentum"], o["nesterov"], f["weight_decay"],
                                f["scale"], f["eps"], o.get("steps", 5))
        assert bool(((m2[i].double() - mom).abs() <= 2.0 ** -23 * (mom.abs() + g[i].double().abs())).all())
        err = float(torch.linalg.norm(w2[i].double() - want))
        assert err <= off + 2.0 ** -22 * (float(torch.linalg.norm(want)) + float(torch.linalg.norm(w[i].double()))), (err, off)
        if copy is not None:
            assert torch.equal(copy[i], w2[i].bfloat16())


def _make(count, rows, cols, dtype, seed=0, ld=None, offset=0, low_rank=False):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + cols)
    ld = ld or cols

    def one(kind, std):
        buf = torch.full((count * rows * ld + offset + 8,), float("nan"), device="cuda", dtype=kind)
        v = buf[offset:offset + count * rows * ld].view(count, rows, ld)[:, :, :cols]
        x = torch.randn(count, rows, cols, device="cuda", generator=g)
        if low_rank:
            x = torch.randn(count, rows, 3, device="cuda", generator=g) @ torch.randn(count, 3, cols, device="cuda", generator=g) + 1e-3 * x
        return v.copy_(x * std)

    return one(torch.float32, 0.05), one(torch.float32, 3e-3), one(dtype, 1e-3)


OPTIONS = dict(lr=0.02, momentum=0.9, weight_decay=0.1, scale=1.3, eps=1e-7)
SHAPES = [(1, 1, 1, None, 0), (2, 1, 40, None, 0), (1, 50, 1, None, 0), (3, 5, 7, 9, 1), (1, 128, 128, None, 0),
          (2, 129, 127, None, 0), (17, 64, 96, None, 0), (1, 256, 256, 260, 4), (2, 300, 700, None, 0), (2, 700, 300, 702, 2),
          (1, 513, 1100, None, 0), (1, 1300, 640, None, 0), (3, 384, 384, None, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count,rows,cols,ld,offset", SHAPES)
def test_update(lm, count, rows, cols, ld, offset, dtype, nesterov):
    w, m, g = _make(count, rows, cols, dtype, ld=ld, offset=offset)
    before = (w.clone(), m.clone(), g)
    copy = torch.empty(count, rows, cols, dtype=torch.bfloat16, device="cuda") if nesterov else None
    lm.muon(w, m, g, nesterov=nesterov, copy=copy, **OPTIONS)
    lm.sync()
    _check(before, (w, m, copy), dict(OPTIONS, nesterov=nesterov))
    # the same bits again, from lists of matrices on another stream
    w3, m3 = list(before[0].clone()), list(before[1].clone())
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        lm.muon(w3, m3, list(g), nesterov=nesterov, **OPTIONS)
        lm.sync()
    assert torch.equal(torch.stack(w3), w) and torch.equal(torch.stack(m3), m)


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(1, 64, 2050), (2, 2047, 70), (1, 515, 2100), (3, 300, 5000), (17, 40, 2000), (1, 2100, 1000), (8, 520, 500),
                                             (2, 1000, 1030), (5, 900, 950)])
def test_forms_of_products(lm, count, rows, cols):
    """Long sums in parts, single CTAs in one and two rounds, pairs."""
    w, m, g = _make(count, rows, cols, torch.float32)
    before = (w.clone(), m.clone(), g)
    lm.muon(w, m, g, **OPTIONS)
    lm.sync()
    _check(before, (w, m, None), dict(OPTIONS, nesterov=True))


@pytest.mark.gpu
@pytest.mark.parametrize("count,rows,cols", [(1, 64, 2050), (3, 300, 500), (2, 1030, 70), (2, 1500, 1600)])
def test_what_the_workspace_held_does_not_matter(lm, count, rows, cols):
    import ctypes as ct
    from tbb_test_b200 import _capi as K
    w, m, g = _make(count, rows, cols, torch.float32)
    need, options, out = ct.c_size_t(), K.MuonOptions(), []
    assert K.lib().b2_muon_workspace(count, rows, cols, ct.byref(need)) == 0
    K.lib().b2_muon_options_default(ct.byref(options))
    for fill in (0, 255):
        space = torch.full((need.value,), fill, dtype=torch.uint8, device="cuda")
        w2, m2 = w.clone(), m.clone()
        lists = [(ct.c_void_p * count)(*[x.data_ptr() for x in xs]) for xs in (w2, m2, g)]
        assert K.lib().b2_muon(count, rows, cols, 0, lists[0], cols, None, 0, lists[1], cols, lists[2], cols, ct.byref(options), space.data_ptr(), need.value,
                               torch.cuda.current_stream().cuda_stream) == 0
        lm.sync()
        out.append((w2, m2))
    assert all(bool(torch.isfinite(x).all()) and torch.equal(x, y) for x, y in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 3, 7])
def test_steps_and_low_rank(lm, steps):
    w, m, g = _make(2, 200, 333, torch.float32, low_rank=True)
    before = (w.clone(), m.clone(), g)
    lm.muon(w, m, g, steps=steps, **OPTIONS)
    _check(before, (w, m, None), dict(OPTIONS, nesterov=True, steps=steps))


@pytest.mark.gpu
def test_even_steps_and_an_update_after_an_update(lm):
    """The buffers end on the other side, and a second call begins from what the first left."""
    w, m, g = _make(2, 333, 200, torch.bfloat16)
    for steps in (2, 4):
        before = (w.clone(), m.clone(), g)
        lm.muon(w, m, g, steps=steps, **OPTIONS)
        _check(before, (w, m, None), dict(OPTIONS, nesterov=True, steps=steps))


@pytest.mark.gpu
def test_in_a_graph(lm):
    w, m, g = _make(2, 200, 130, torch.float32)
    w1, m1 = w.clone(), m.clone()
    for _ in range(2):
        lm.muon(w1, m1, g, **OPTIONS)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lm.muon(w, m, g, **OPTIONS)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w, w1) and torch.equal(m, m1)


@pytest.mark.gpu
def test_singular_values_come_near_one(lm):
    g = torch.Generator(device="cuda").manual_seed(3)
    u, v = (torch.linalg.qr(torch.randn(n, 200, device="cuda", generator=g).double())[0] for n in (300, 200))
    s = torch.logspace(0, -1.5, 200, device="cuda", dtype=torch.float64)
    grad = ((u * s) @ v.T).float()
    w, m = torch.zeros(1, 300, 200, device="cuda"), torch.zeros(1, 300, 200, device="cuda")
    lm.muon(w, m, grad[None], lr=1.0, momentum=0.0, nesterov=False)
    s = torch.linalg.svdvals(-w[0].double())
    assert 0.65 <= float(s.min()) and float(s.max()) <= 1.21


@pytest.mark.gpu
def test_zero_gradient_and_scales(lm):
    w = torch.randn(2, 70, 90, device="cuda")
    m, g = torch.zeros_like(w), torch.zeros_like(w)
    before = w.clone()
    lm.muon(w, m, g, lr=0.5, weight_decay=0.25)
    assert torch.equal(w, before * 0.875) and not m.any()
    for k in (1e-25, 1e25):  # x does not depend on the gradient's scale (and eps is far below or above the norm)
        g = torch.randn(1, 100, 130, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * k
        w, m = torch.zeros_like(g), torch.zeros_like(g)
        lm.muon(w, m, g, lr=1.0, eps=0.0)
        want, _, off = _exact(torch.zeros(100, 130, device="cuda", dtype=torch.float64), 0.0, g[0].double(), 1.0, float(np.float32(0.95)), True, 0.0, 1.0, 0.0)
        assert float(torch.linalg.norm(w[0].double() - want)) <= off + 2.0 ** -22 * float(torch.linalg.norm(want))


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(70, 90), (33, 17)])
def test_without_eps(lm, rows, cols, dtype, nesterov):
    """A matrix of zeros beside others; gradients as small and as large as fp32 has them, whose norms' reciprocals it has not."""
    g = torch.randn(5, rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    g[1] = 0.0
    g[2] *= 2.0 ** -124
    g[3] = 0.0
    g[3, 5, 7] = 2.0 ** -133  # exact in either type, and |u| is this number alone
    g[4] *= 2.0 ** 124
    w, m = torch.randn(5, rows, cols, device="cuda"), torch.zeros(5, rows, cols, device="cuda")
    before = w.clone()
    o = dict(lr=0.5, weight_decay=0.25, eps=0.0, momentum=0.0, nesterov=nesterov)
    lm.muon(w, m, g, **o)
    assert torch.equal(w[1], before[1] * 0.875) and not m[1].any()
    for i in (0, 2, 3, 4):
        want, _, off = _exact(before[i].double(), 0.0, g[i].double(), 0.5, 0.0, nesterov, 0.25, 1.0, 0.0)
        assert float(torch.linalg.norm(w[i].double() - want)) <= off + 2.0 ** -22 * (float(torch.linalg.norm(want)) + float(torch.linalg.norm(before[i])))


@pytest.mark.gpu
def test_not_a_number_stays_in_its_matrix(lm):
    w, m, g = _make(3, 130, 260, torch.float32)
    before = (w.clone(), m.clone(), g.clone())
    g[1, 4, 5] = float("nan")
    lm.muon(w, m, g, nesterov=True, **OPTIONS)
    assert bool(torch.isnan(w[1]).all())
    pick = lambda t: t[::2]  # noqa: E731
    _check(tuple(map(pick, before)), (pick(w), pick(m), None), dict(OPTIONS, nesterov=True))


@pytest.mark.gpu
def test_wrapper_refuses(lm):
    x = torch.zeros(2, 8, 16, device="cuda")
    for call in (lambda: lm.muon(x, x, x.half(), lr=1), lambda: lm.muon(x.bfloat16(), x, x, lr=1), lambda: lm.muon(x, x[:1], x, lr=1),
                 lambda: lm.muon(x, x, x[:, :4], lr=1), lambda: lm.muon(x, x, x, lr=1, copy=x), lambda: lm.muon([], [], [], lr=1),
                 lambda: lm.muon(x.mT, x.mT, x.mT, lr=1), lambda: lm.muon(x.cpu(), x.cpu(), x.cpu(), lr=1)):
        with pytest.raises(ValueError):
            call()


def test_c_entry_refuses_before_any_device_work(native):
    import ctypes as ct
    from tbb_test_b200 import _capi as K
    lib = K.lib()
    o = K.MuonOptions()
    assert lib.b2_muon_options_default(ct.byref(o)) == K.OK and o.steps == 5 and o.nesterov == 1
    assert lib.b2_muon_options_default(None) == K.ERR_INVALID
    two = (ct.c_void_p * 2)(256, 512)
    good = dict(count=2, rows=4, cols=8, dtype=0, w=two, ldw=8, copy=None, ldc=0, m=two, ldm=8, g=two, ldg=8, o=ct.byref(o), ws=ct.c_void_p(256),
                ws_bytes=1 << 30, stream=None)

    def muon(**kw):
        return lib.b2_muon(*{**good, **kw}.values())

    def options(**kw):
        x = K.MuonOptions()
        lib.b2_muon_options_default(ct.byref(x))
        for k, v in kw.items():
            setattr(x, k, v)
        return ct.byref(x)

    for kw in (dict(count=-1), dict(rows=0), dict(cols=65537), dict(dtype=2), dict(w=None), dict(m=None), dict(g=None), dict(o=None), dict(ws=None),
               dict(ldw=7), dict(ldm=7), dict(ldg=7), dict(copy=two, ldc=7), dict(ws=ct.c_void_p(100)), dict(ws_bytes=10),
               dict(w=(ct.c_void_p * 2)(256, None)), dict(m=(ct.c_void_p * 2)(256, 514)), dict(copy=(ct.c_void_p * 2)(256, 257), ldc=8),
               dict(o=options(steps=0)), dict(o=options(steps=101)), dict(o=options(eps=float("nan"))), dict(o=options(eps=-1.0))):
        assert muon(**kw) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
    assert muon(count=0, w=None, m=None, g=None, ws=None) == K.OK
    need = ct.c_size_t()
    assert lib.b2_muon_workspace(2, 4, 8, ct.byref(need)) == K.OK and need.value > 0
    assert lib.b2_muon_workspace(2, 4, 8, None) == K.ERR_INVALID
