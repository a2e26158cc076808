"""Embedding rows and the table's gradient (tbb_test_b200.lm) against the formulas in 64 bits.

Tolerances, fixed by the arithmetic: one fp32 product and one rounding for a row; for a gradient element of k terms any
order of fp32 additions is within k * 2^-24 of the sum of magnitudes, one more rounding for the scale, and outputs
add the unit roundoff of their type."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = {k: torch.finfo(v).eps / 2 for k, v in DTYPE.items()}  # unit roundoff: 2^-24, 2^-8


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _tokens(n, vocab, kind, seed, dtype=torch.int64):
    r = np.random.RandomState(seed)
    if kind == "same":
        t = np.full(n, vocab - 1)
    elif kind == "zipf":
        t = np.minimum(np.exp(r.rand(n) * np.log(vocab + 1)).astype(np.int64) - 1, vocab - 1)
    elif kind == "padding":
        t = np.full(n, -1)
        t[::5] = r.randint(0, vocab, len(t[::5]))
        t[1::5] = vocab
        t[2::5] = -2 ** 31
        t[3::5] = 2 ** 31 - 1
    elif kind == "none":
        t = np.full(n, vocab + 3)
    else:
        t = r.randint(0, vocab, n)
    return torch.tensor(t, dtype=dtype, device="cuda")


def _rows(n, d, dtype, seed, ld=None, offset=0):
    """n x d values, as a view into a buffer with other rows and columns of NaN around it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or d
    buf = torch.full((n * ld + offset + 8,), float("nan"), device="cuda", dtype=DTYPE[dtype])
    view = buf[offset:offset + n * ld].view(n, ld)[:, :d]
    view.copy_(torch.randn(n, d, device="cuda", generator=g))
    return view


# (width, leading dimension, offset in elements): whole 16-byte pieces, narrower vectors, single elements
LAYOUTS = [(512, 512, 0), (128, 136, 0), (36, 44, 4), (30, 34, 2), (7, 9, 1), (1, 1, 0), (2500, 2504, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("width,ld,offset", LAYOUTS)
@pytest.mark.parametrize("n,vocab,kind", [(1, 1, "any"), (77, 50, "padding"), (3000, 4001, "any")])
def test_embed(lm, dtype, width, ld, offset, n, vocab, kind):
    t = _tokens(n, vocab, kind, 1, torch.int32 if width % 2 else torch.int64)
    table = _rows(vocab, width, dtype, 2, ld, offset)
    out = _rows(n, width, dtype, 3, ld, offset)
    assert lm.embed(t, table, scale=1.7, out=out) is out
    t, x = t.cpu().long(), table.double().cpu()
    ok = (t >= 0) & (t < vocab)
    want = torch.where(ok[:, None], x[t.clamp(0, vocab - 1)] * float(np.float32(1.7)), 0.0)
    err = (out.double().cpu() - want).abs()
    assert bool((err <= want.abs() * (2.0 ** -24 + EPS[dtype])).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n,vocab,width,ld,offset,kind", [
    (1, 1, 8, 8, 0, "any"), (1, 300, 512, 512, 0, "any"), (9, 3, 5, 7, 1, "any"), (1000, 10007, 203, 203, 0, "zipf"),
    (1000, 7, 64, 72, 0, "any"), (777, 64, 36, 44, 4, "padding"), (300, 20, 16, 16, 0, "none"), (8192, 100, 40, 40, 0, "zipf"),
    (8193, 1000, 24, 24, 0, "zipf"), (8200, 70000, 8, 8, 0, "any"), (30001, 70000, 130, 136, 0, "zipf"),
    (50000, 5, 64, 64, 0, "same"), (50000, 1 << 21, 2, 2, 0, "any"), (300000, 257, 8, 8, 0, "zipf"), (20000, 3000, 1100, 1100, 0, "padding")])
def test_embed_grad(lm, dtype, n, vocab, width, ld, offset, kind):
    t = _tokens(n, vocab, kind, n, torch.int64 if width % 3 else torch.int32)
    dout = _rows(n, width, dtype, 5, ld, offset)
    out = _rows(vocab, width, dtype, 6, ld, offset)
    assert lm.embed_grad(t, dout, vocab, scale=0.3, out=out) is out
    again = lm.embed_grad(t, dout, vocab, scale=0.3)
    assert torch.equal(out, again)  # the same bits, whatever ran where
    x = dout.double().cpu()
    t = t.cpu().long()
    ok = (t >= 0) & (t < vocab)
    s = float(np.float32(0.3))
    want = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, t[ok], x[ok] * s)
    size = torch.zeros(vocab, width, dtype=torch.float64).index_add_(0, t[ok], x[ok].abs() * s)
    terms = torch.bincount(t[ok], minlength=vocab)[:, None].double()
    err = (out.double().cpu() - want).abs()
    assert bool((err <= size * (terms + 1) * 2.0 ** -24 + want.abs() * EPS[dtype] * 1.01).all())


@pytest.mark.gpu
def test_gradient_is_the_lookups_transpose(lm):
    """<dout, embed(x)> = <embed_grad(dout), x> for any x: the lookup is linear in the table."""
    t = _tokens(5000, 800, "padding", 3)
    x, dout = _rows(800, 96, "fp32", 1), _rows(5000, 96, "fp32", 2)
    a = (dout.double() * lm.embed(t, x, scale=2.0).double()).sum()
    b = (lm.embed_grad(t, dout, 800, scale=2.0).double() * x.double()).sum()
    assert abs(float(a - b)) <= 5000 * 2.0 ** -24 * float((dout.abs().sum(1) * 2.0 * 5).double().sum())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["padding", "zipf"])
def test_gradient_is_the_lookups_transpose_in_large_products(lm, kind):
    """The same with positive values, so that the products are large against what they may be off: one rounding per row of the lookup, and per
    element of the gradient an addition for each of its terms and the scale."""
    n, vocab = 5000, 800
    t = _tokens(n, vocab, kind, 3)
    x, dout = _rows(vocab, 96, "fp32", 1).abs(), _rows(n, 96, "fp32", 2).abs()
    a = (dout.double() * lm.embed(t, x, scale=2.0).double()).sum()
    b = (lm.embed_grad(t, dout, vocab, scale=2.0).double() * x.double()).sum()
    ok = (t >= 0) & (t < vocab)
    terms = int(torch.bincount(t[ok].cpu(), minlength=vocab).max())
    size = float((dout[ok].double() * x[t[ok]].double() * 2.0).sum())
    bound = (terms + 2) * 2.0 ** -24 * size
    assert bound < size * 1e-3 and abs(float(a - b)) <= bound


@pytest.mark.gpu
def test_nan_and_inf_stay_in_their_rows(lm):
    t = torch.tensor([0, 1, -1, 1, 2], device="cuda")
    dout = torch.ones(5, 64, device="cuda")
    dout[2] = float("nan")  # padding: takes no part
    dout[4, 3] = float("inf")
    g = lm.embed_grad(t, dout, 4)
    want = torch.tensor([1.0, 2.0, 1.0, 0.0], device="cuda")[:, None].expand(4, 64).clone()
    want[2, 3] = float("inf")
    assert torch.equal(g, want)


@pytest.mark.gpu
def test_on_another_stream_and_without_tokens(lm):
    s = torch.cuda.Stream()
    table = _rows(64, 32, "fp32", 1)
    t = _tokens(20000, 64, "any", 1)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = lm.embed(t, table)
        g = lm.embed_grad(t, y, 64)
    s.synchronize()
    count = torch.bincount(t, minlength=64)[:, None]
    assert torch.allclose(g, table * count, rtol=1e-5)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert lm.embed(none, table).shape == (0, 32)
    assert not lm.embed_grad(none, table[:0], 64).any()


@pytest.mark.gpu
def test_in_a_graph(lm):
    table = _rows(500, 64, "bf16", 1)
    t = _tokens(20000, 500, "zipf", 1)
    y = lm.embed(t, table)
    want = lm.embed_grad(t, y, 500)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lm.embed(t, table)
        got = lm.embed_grad(t, out, 500)
    out.zero_()
    got.zero_()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, y) and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("n", range(1, 10))
def test_few_tokens_end_behind_their_sums(lm, n, graph):
    """Up to eight tokens are one chunk, whose runs nothing joins. What follows on the stream finds whole sums, and may write over the
    gradient's input and the workspace."""
    import ctypes as C
    from tbb_test_b200 import _capi as K
    vocab, width = 40, 8192
    t = _tokens(n, vocab, "any", n)
    dout = _rows(n, width, "fp32", n)
    want = torch.zeros(vocab, width, device="cuda", dtype=torch.float64).index_add_(0, t, dout.double())
    size = torch.zeros(vocab, width, device="cuda", dtype=torch.float64).index_add_(0, t, dout.double().abs())
    kept, out, need = dout.clone(), torch.empty(vocab, width, device="cuda"), C.c_size_t()
    assert K.lib().b2_embed_grad_workspace(n, vocab, width, C.byref(need)) == K.OK
    space, got = torch.empty(need.value, dtype=torch.uint8, device="cuda"), torch.empty_like(out)

    def call():
        dout.copy_(kept)
        assert K.lib().b2_embed_grad(t.data_ptr(), 8, n, dout.data_ptr(), 0, width, vocab, width, 1.0, out.data_ptr(), width, space.data_ptr(),
                                     space.numel(), torch.cuda.current_stream().cuda_stream) == K.OK
        got.copy_(out)
        dout.fill_(float("nan"))
        space.fill_(255)
        out.fill_(float("nan"))

    call()
    torch.cuda.synchronize()
    run = call
    if graph:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        run = g.replay
    for _ in range(20):
        got.zero_()
        run()
        assert bool(((got.double() - want).abs() <= size * (n + 1) * 2.0 ** -24 + want.abs() * EPS["fp32"] * 1.01).all())


@pytest.mark.gpu
def test_wrapper_refuses(lm):
    table = torch.zeros(8, 16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: lm.embed(t.float(), table), lambda: lm.embed(t.cpu(), table), lambda: lm.embed(t, table.half()),
                 lambda: lm.embed(t, table.t()), lambda: lm.embed(t, table[0]), lambda: lm.embed(t, table, out=table),
                 lambda: lm.embed_grad(t, table, 8), lambda: lm.embed_grad(t, table[:4], 8, out=table[:7]),
                 lambda: lm.embed_grad(t, table[:4].cpu(), 8)):
        with pytest.raises(ValueError):
            call()


def test_c_entries_refuse_before_any_device_work(native):
    """Bad arguments come back as B2_ERR_INVALID with a text, with or without a GPU."""
    import ctypes as C
    from tbb_test_b200 import _capi as K
    lib, p = K.lib(), C.c_void_p(256)
    good = dict(tokens=p, size=4, n=3, table=p, dtype=0, vocab=5, width=8, ld=8, scale=1.0, out=p, ldo=8, stream=None)

    def embed(**kw):
        return lib.b2_embed(*{**good, **kw}.values())

    grad = dict(tokens=p, size=4, n=3, dout=p, dtype=0, ld=8, vocab=5, width=8, scale=1.0, out=p, ldo=8, ws=p, ws_bytes=1 << 20, stream=None)

    def embed_grad(**kw):
        return lib.b2_embed_grad(*{**grad, **kw}.values())

    for kw in (dict(size=2), dict(dtype=2), dict(width=0), dict(vocab=0), dict(ld=7), dict(ldo=7), dict(tokens=None), dict(out=None),
               dict(n=1 << 31), dict(vocab=1 << 31)):
        assert embed(**kw) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
        assert embed_grad(**kw) == K.ERR_INVALID, kw
    assert embed_grad(ws=None) == K.ERR_INVALID
    assert embed_grad(ws=C.c_void_p(264)) == K.ERR_INVALID
    assert embed_grad(ws_bytes=16) == K.ERR_INVALID and b"workspace" in lib.b2_last_error(None)
    assert embed_grad(size=8, tokens=C.c_void_p(260)) == K.ERR_INVALID
    need = C.c_size_t()
    assert lib.b2_embed_grad_workspace(1000, 50, 64, C.byref(need)) == K.OK and need.value > 0
    assert lib.b2_embed_grad_workspace(1000, 50, 64, None) == K.ERR_INVALID
    assert embed(n=0, tokens=None, out=None) == K.OK  # nothing to do


def test_no_device_is_an_error(native):
    import ctypes as C
    from conftest import HAS_GPU
    if HAS_GPU:
        pytest.skip("a GPU is present")
    from tbb_test_b200 import _capi as K
    p = C.c_void_p(256)
    assert K.lib().b2_embed(p, 4, 3, p, 0, 5, 8, 8, 1.0, p, 8, None) == K.ERR_CUDA
    assert b"no CPU path" in K.lib().b2_last_error(None)
