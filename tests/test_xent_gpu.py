"""Cross entropy over a vocabulary (tbb_test_b200.lm.xent) against the formulas in 64 bits, element by element.

Tolerances, from the arithmetic: a sum of k products in the tensor core takes k / 16 additions, each off by at most 2^-23
of the sum of magnitudes; exp and log add a few units of 2^-23; d, the logits' gradient, is rounded to its type once (bf16
2^-8, fp16 pairs 2^-20 with room, but nothing finer than 2^-50; nothing
in fp32 is finer than 2^-126), and so are the outputs. Errors of d go through the two
products in magnitude."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}
ULP = 2.0 ** -23


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _matrix(rows, cols, dtype, g, std, ld=None, offset=0):
    """rows x cols normal values as a view into a buffer that is NaN elsewhere."""
    ld = ld or cols
    buf = torch.full((rows * ld + offset + 8,), float("nan"), device="cuda", dtype=DTYPE[dtype])
    view = buf[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(torch.randn(rows, cols, device="cuda", generator=g) * std)
    return view


def _case(rows, width, vocab, dtype, seed=0, padding=0.2, ldh=None, ldw=None, offset=0, peak=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + width)
    w = _matrix(vocab, width, dtype, g, 2.0 * width ** -0.5, ldw, offset)
    h = _matrix(rows, width, dtype, g, 1.0, ldh, offset)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    h.copy_((h.float() + w[t].float() * peak * torch.rand(rows, 1, device="cuda", generator=g)).to(h.dtype))
    pad = torch.rand(rows, device="cuda", generator=g) < padding
    t[pad] = -100
    return h, w, t


def _check(h, w, t, scale, got, dtype):
    vocab, width = w.shape
    ok = (t >= 0) & (t < vocab)
    h, w, at = h[ok].double(), w.double(), t[ok].long()
    rows = torch.arange(len(at), device="cuda")
    x = h @ w.T
    size = (h.abs() @ w.abs().T).amax(1) if len(at) else torch.zeros(0, device="cuda", dtype=torch.float64)
    lse = torch.logsumexp(x, 1)
    loss, dh, dw = got if isinstance(got, tuple) else (got, None, None)
    want = lse - x[rows, at]
    off = 2 * (width / 16 + 8) * ULP * size  # of a difference of two logits
    assert bool((loss[~ok] == 0).all())
    assert bool(((loss[ok].double() - want).abs() <= off + 8 * ULP * (1 + lse.abs() + x[rows, at].abs())).all())
    if dh is None:
        return
    p = torch.exp(x - lse[:, None])
    d = p.clone()
    d[rows, at] -= 1.0
    unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -20
    out = torch.finfo(DTYPE[dtype]).eps / 2
    err = p * (torch.expm1(off)[:, None] + 16 * ULP) + d.abs() * unit + (2.0 ** -126 if dtype == "bf16" else 2.0 ** -50)
    s = abs(scale)
    assert not dh[~ok].any()
    want = d @ w * scale
    bound = s * (err @ w.abs() + (vocab / 16 + 8) * ULP * (d.abs() @ w.abs())) + want.abs() * out * 1.01
    assert bool(((dh[ok].double() - want).abs() <= bound).all())
    want = d.T @ h * scale
    bound = s * (err.T @ h.abs() + (len(at) / 16 + 8) * ULP * (d.abs().T @ h.abs())) + want.abs() * out * 1.01
    assert bool(((dw.double() - want).abs() <= bound).all())


# rows, width, vocab, ldh, ldw, offset: one element to several tiles and pieces; rows that are no whole 16-byte pieces
SHAPES = [
    (1, 1, 1, None, None, 0), (1, 8, 300, None, None, 0), (3, 64, 2, None, None, 0), (5, 7, 31, 9, 11, 1),
    (96, 512, 10007, None, None, 0), (255, 72, 257, None, 80, 0), (256, 128, 256, None, None, 0),
    (257, 200, 513, 208, 208, 8), (300, 203, 1000, None, None, 0), (700, 136, 3001, 140, 144, 4), (1030, 1100, 2100, None, None, 0),
    (2, 2056, 5000, None, None, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,vocab,ldh,ldw,offset", SHAPES)
def test_losses_and_gradients(lm, dtype, rows, width, vocab, ldh, ldw, offset):
    h, w, t = _case(rows, width, vocab, dtype, ldh=ldh, ldw=ldw, offset=offset)
    if rows == 1:
        t[0] = vocab - 1
    g = torch.Generator(device="cuda").manual_seed(1)
    dh, dw = _matrix(rows, width, dtype, g, 1.0, ldh, offset), _matrix(vocab, width, dtype, g, 1.0, ldw, offset)
    got = lm.xent(h, w, t, scale=0.37, dh=dh, dw=dw)
    lm.sync()
    assert got[1] is dh and got[2] is dw
    _check(h, w, t, float(np.float32(0.37)), got, dtype)
    only = lm.xent(h, w, t.int(), grad=False)
    assert torch.equal(only, got[0])
    again = lm.xent(h, w, t, scale=0.37)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_several_pieces(lm, dtype):
    """More rows x vocabulary than one piece of the logits' gradients holds."""
    rows, vocab = (12000, 30001) if dtype == "bf16" else (6000, 30001)
    h, w, t = _case(rows, 64, vocab, dtype)
    _check(h, w, t, 1.0, lm.xent(h, w, t), dtype)
    lm.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,vocab", [(1200, 72, 90), (32768, 8, 5), (32769, 24, 70), (70001, 40, 33)])
def test_many_rows(lm, dtype, rows, width, vocab):
    """More rows than blocks that list them, and than every block counts by itself."""
    h, w, t = _case(rows, width, vocab, dtype)
    t[: rows // 3] = -100
    _check(h, w, t, 1.0, lm.xent(h, w, t), dtype)
    lm.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,vocab", [(1, 3973, 806), (23, 2000, 9472), (290, 1100, 130), (297, 1100, 130), (64, 1500, 1), (130, 2049, 4099), (1100, 900, 1200)])
def test_few_tiles(lm, dtype, rows, width, vocab):
    """Long sums in parts and whole, with gradients and without."""
    h, w, t = _case(rows, width, vocab, dtype)
    got = lm.xent(h, w, t)
    _check(h, w, t, 1.0, got, dtype)
    assert torch.equal(lm.xent(h, w, t, grad=False), got[0])
    t[:] = -100
    loss, dh, dw = lm.xent(h, w, t)
    assert not loss.any() and not dh.any() and not dw.any()
    lm.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,width,vocab", [
    ("bf16", 10, 8, 1400001), ("fp32", 20, 8, 700001),  # few rows: logits are kept, d goes in pieces
    ("bf16", 600, 2048, 30001), ("fp32", 300, 264, 60002),  # kept although they are more than the L2 cache should hold
    ("bf16", 3000, 200, 6001), ("fp32", 3000, 200, 6003)])  # too many: computed a second time
def test_logits_kept_or_computed_again(lm, dtype, rows, width, vocab):
    h, w, t = _case(rows, width, vocab, dtype)
    _check(h, w, t, 1.0, lm.xent(h, w, t), dtype)
    lm.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,vocab", [(1, 8, 300), (5, 1500, 700), (70, 200, 1000), (300, 100, 3001), (300, 64, 40000), (3000, 200, 6003)])
def test_what_the_workspace_held_does_not_matter(lm, dtype, rows, width, vocab):
    """NaN everywhere, in every type, against zeros: equal bits."""
    import ctypes as ct
    from tbb_test_b200 import _capi as K
    h, w, t = _case(rows, width, vocab, dtype)
    kind, out = 1 if dtype == "bf16" else 0, []
    need = ct.c_size_t()
    assert K.lib().b2_xent_workspace(rows, width, vocab, kind, 1, w.data_ptr(), width, ct.byref(need)) == 0
    for fill in (0, 255):
        space = torch.full((need.value,), fill, dtype=torch.uint8, device="cuda")
        loss, dh, dw = torch.zeros(rows, device="cuda"), torch.zeros_like(h), torch.zeros_like(w)
        assert K.lib().b2_xent(rows, width, vocab, kind, h.data_ptr(), width, w.data_ptr(), width, t.data_ptr(), 8, 1.0, loss.data_ptr(), dh.data_ptr(),
                               width, dw.data_ptr(), width, space.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream) == 0
        lm.sync()
        out.append((loss, dh, dw))
    assert all(bool(torch.isfinite(x).all()) and torch.equal(x, y) for x, y in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_rows_without_a_target(lm, dtype):
    """They cost nothing and nothing of them gets out, not even NaN; a call of such rows alone gives zeros."""
    h, w, t = _case(500, 96, 700, dtype, padding=0.0)
    t[::3] = 700
    t[1] = 2 ** 40
    t[2] = -1
    bad = (t < 0) | (t >= 700)
    clean = lm.xent(h, w, t, scale=0.01)
    h[bad] = float("nan")
    h[0] = float("inf")
    got = lm.xent(h, w, t, scale=0.01)
    assert all(torch.equal(a, b) for a, b in zip(clean, got))
    _check(torch.where(bad[:, None], 0.0, h.float()).to(h.dtype), w, t, 0.01, got, dtype)
    loss, dh, dw = lm.xent(h, w, torch.full_like(t, -100))
    assert not loss.any() and not dh.any() and not dw.any()
    loss, dh, dw = lm.xent(h[:0], w, t[:0])
    assert loss.shape == (0,) and dh.shape == (0, 96) and dw.shape == w.shape and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_large_and_infinite_logits(lm, dtype):
    h, w, t = _case(64, 32, 900, dtype, padding=0.0)
    _check(h * 200, w, t, 1.0, lm.xent(h * 200, w, t), dtype)  # softmax at its corners: p is 0 or 1
    _check(h * 0, w, t, 1.0, lm.xent(h * 0, w, t), dtype)  # all logits equal
    w[5] = float("nan")  # a weight that is not finite reaches every row
    loss, dh, dw = lm.xent(h, w, t)
    assert bool(torch.isnan(loss).all())
    lm.sync()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e20])
def test_infinity_stays_in_its_row_fp32(lm, size):
    """One infinite element of h must not set the scale that the other rows are split with."""
    h, w, t = _case(50, 40, 300, "fp32", padding=0.0)
    h, w = h * size, w / size
    clean = lm.xent(h, w, t)
    h[7, 3] = float("inf")
    loss, dh, _ = lm.xent(h, w, t)
    rest = torch.arange(50, device="cuda") != 7
    assert bool(torch.isnan(loss[7])) and torch.equal(loss[rest], clean[0][rest])
    assert torch.equal(dh[rest], clean[1][rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,width,vocab", [(64, 32, 900), (5, 1500, 700), (300, 64, 40000), (3000, 200, 6003), (2, 2056, 5000)])
def test_infinite_weights(lm, dtype, rows, width, vocab):
    """A logit of -inf is a probability of 0, and only the columns of dh that its weight's infinity stands in are NaN (0 times infinity)."""
    h, w, t = _case(rows, width, vocab, dtype, padding=0.0)
    a, b = 3, width - 2
    h[:, a], h[:, b] = 1.0, -0.5
    h[-1, a] = 1e-20  # far below what the pair of fp16 matrices holds beside the others, but not 0
    out = torch.tensor([7, vocab // 2, vocab - 1], device="cuda")
    t[(t[:, None] == out).any(1)] = 8
    for v, c, x in zip(out.tolist(), (a, b, a), (float("-inf"), float("inf"), float("-inf"))):
        w[v, c] = x
    got = lm.xent(h, w, t, scale=0.5)
    lm.sync()
    assert torch.equal(lm.xent(h, w, t, grad=False), got[0])
    # what a vocabulary without those words gives
    keep = torch.ones(vocab, dtype=torch.bool, device="cuda")
    keep[out] = False
    place = torch.cumsum(keep, 0) - 1
    loss, dh, dw = got
    assert bool(torch.isnan(dh[:, [a, b]]).all()) and not dw[out].any()
    rest = torch.ones(width, dtype=torch.bool, device="cuda")
    rest[[a, b]] = False
    some = dh.clone()
    x = h.double() @ w[keep].double().T
    d = torch.softmax(x, 1)
    d[torch.arange(rows, device="cuda"), place[t]] -= 1.0
    some[:, ~rest] = (0.5 * d @ w[keep].double())[:, ~rest].to(dh.dtype)
    _check(h, w[keep], place[t], 0.5, (loss, some, dw[keep]), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_infinite_weights_by_sign(lm, dtype):
    """+inf in a row's logits, and 0 times infinity, make its loss NaN; the target's -inf makes it +inf."""
    h, w, t = _case(40, 64, 500, dtype, padding=0.0)
    t[:] = 3
    t[5] = 11
    w[11, 9] = float("-inf")
    h[:, 9] = 0.25
    h[1, 9], h[2, 9], h[3, 9] = -0.25, 0.0, -1e-20
    loss = lm.xent(h, w, t, grad=False)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[1:4] = True
    assert bool(torch.isnan(loss[bad]).all()) and float(loss[5]) == float("inf")
    bad[5] = True
    assert bool(torch.isfinite(loss[~bad]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,vocab", [(300, 2000, 60002), (2100, 4096, 65536), (300, 2048, 1000), (300, 1024, 60002)])
def test_nearly_certain_targets(lm, rows, width, vocab):
    """Logits of 65 whose target has a probability of about 1 - 1e-4, kept and computed again: dh relative to its own rows. The logits of a row
    come from one and the same sums in both passes, so p adds up to 1 and d is off by its share of two things only: its rounding to bf16, and
    what the sums of 16 k-blocks (64 additions of the tensor core, each at 2^-23 of the magnitudes) and their join are off."""
    g = torch.Generator(device="cuda").manual_seed(width)
    common = torch.randn(width, device="cuda", generator=g)
    common *= 3.0 / torch.linalg.norm(common)
    own = torch.randn(vocab, width, device="cuda", generator=g) * (2.0 * width ** -0.5)
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    w, h = (common + own).bfloat16(), (5.0 * common + 5.0 * own[t]).bfloat16()
    del own
    _, dh, _ = lm.xent(h, w, t)
    lm.sync()
    hd, wd, at = h.double(), w.double(), torch.arange(rows, device="cuda")
    x = hd @ wd.T
    size = float((hd.abs() @ wd.abs().T).max())
    d = torch.softmax(x, 1)
    assert 1e-6 < float((1.0 - d[at, t]).median()) < 1e-2 and float(x[at, t].median()) > 55.0
    d[at, t] -= 1.0
    off = 2 * (64 + width / 1024 + 8) * ULP * size
    bound = (np.expm1(off) + 2.0 ** -8 + 2.0 ** -8) * d.abs().sum(1) * float(torch.linalg.norm(wd, dim=1).max()) + 2.0 ** -20 * float(torch.linalg.norm(wd, dim=1).max())
    assert bool((torch.linalg.norm(dh.double() - d @ wd, dim=1) <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,vocab", [(300000, 64, 64), (300000, 200, 70), (300003, 63, 64), (1 << 20, 64, 64)])
def test_sums_over_many_rows_have_no_bias(lm, rows, width, vocab):
    """dw of words that are never the target: every term is positive. A sum of n truncating additions is too small by up to n 2^-24 of itself in the
    mean; with sums of 512 k-blocks at most (2048 additions) that is 1.2e-4. The roundings to bf16, of d and of dw, have no sign: d's are spread
    over all rows; dw's, of up to 2^-8 and 2^-8 / sqrt(3) in the mean square, over the n elements looked at, four times their mean for a bound."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = (torch.rand(rows, width, device="cuda", generator=g) + 0.5).bfloat16()
    w = (torch.randn(vocab, width, device="cuda", generator=g) * 0.05).bfloat16()
    t = torch.randint(0, 4, (rows,), device="cuda", generator=g)
    _, _, dw = lm.xent(h, w, t, scale=1.0 / rows)
    lm.sync()
    want = torch.zeros(vocab, width, device="cuda", dtype=torch.float64)
    for part, at in zip(h.split(1 << 18), t.split(1 << 18)):
        d = torch.softmax(part.double() @ w.double().T, 1)
        d[torch.arange(len(at), device="cuda"), at] -= 1.0
        want += d.T @ part.double() / rows
    off = ((dw.double() - want) / want)[4:]
    # a word's probability is nearly the same in all rows, and with it the rounding of d: 2^-8 / sqrt(3) over the words
    bound = 1.2e-4 + 4 * 2.0 ** -8 / 3 ** 0.5 * ((vocab - 4) ** -0.5 + off.numel() ** -0.5)
    assert abs(float(off.mean())) <= bound


@pytest.mark.gpu
def test_sums_over_a_long_vocabulary_have_no_bias(lm):
    """dh of rows with positive weights: the sum of p w is positive; as above, 2048 additions at most."""
    rows, width, vocab = 2048, 1024, 1 << 17
    g = torch.Generator(device="cuda").manual_seed(5)
    h = (torch.randn(rows, width, device="cuda", generator=g) * 0.1).bfloat16()
    w = (torch.rand(vocab, width, device="cuda", generator=g) + 0.5).bfloat16()
    _, dh, _ = lm.xent(h, w, torch.zeros(rows, dtype=torch.int64, device="cuda"))
    lm.sync()
    total = torch.zeros(rows, device="cuda", dtype=torch.float64)
    want = torch.zeros(rows, width, device="cuda", dtype=torch.float64)
    for part in w.split(1 << 14):
        p = torch.exp(h.double() @ part.double().T)
        total += p.sum(1)
        want += p @ part.double()
    want /= total[:, None]
    off = (dh.double() - want + w[0].double()) / want
    # the roundings of d are spread over the vocabulary, those of dh over all its elements
    assert abs(float(off.mean())) <= 1.2e-4 + 4 * 2.0 ** -8 / 3 ** 0.5 * (vocab ** -0.5 + off.numel() ** -0.5)


@pytest.mark.gpu
def test_small_and_large_magnitudes_fp32(lm):
    """The split of fp32 matrices follows their largest element."""
    for a, b in ((1e-20, 1e20), (1e15, 1e-15), (1e-30, 1.0)):
        h, w, t = _case(70, 40, 500, "fp32", padding=0.0)
        h, w = h * a, w * b
        _check(h, w, t, 1.0, lm.xent(h, w, t), "fp32")


@pytest.mark.gpu
def test_gradients_against_differences(lm):
    h, w, t = _case(40, 24, 70, "fp32")
    g = torch.Generator(device="cuda").manual_seed(9)
    loss, dh, dw = lm.xent(h, w, t, scale=1.0)
    for x, d in ((h, dh), (w, dw)):
        step = torch.randn(x.shape, device="cuda", generator=g)
        eps = 2.0 ** -7

        def total(k):
            a = x + k * eps * step
            return lm.xent(a if x is h else h, a if x is w else w, t, grad=False).double().sum()

        # fourth-order difference: truncation eps^4 of a function whose scale is 1, losses at 2^-22 of their sum
        slope = (8 * (total(1) - total(-1)) - (total(2) - total(-2))) / (12 * eps)
        want = (d.double() * step.double()).sum()
        size = float((d.double().abs() * step.double().abs()).sum())
        assert abs(float(slope - want)) <= 2.0 ** -10 * size + 2.0 ** -20 * float(loss.double().sum()) / eps


@pytest.mark.gpu
def test_one_gradient_only_and_another_stream(lm):
    from tbb_test_b200 import _capi as K
    import ctypes as C
    h, w, t = _case(300, 64, 800, "bf16")
    loss, dh, dw = lm.xent(h, w, t, scale=0.5)
    need = C.c_size_t()
    assert K.lib().b2_xent_workspace(300, 64, 800, 1, 1, w.data_ptr(), 64, C.byref(need)) == K.OK
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        for which in (0, 1):
            row, out = torch.empty_like(loss), torch.empty_like(dw if which else dh)
            rc = K.lib().b2_xent(300, 64, 800, 1, h.data_ptr(), 64, w.data_ptr(), 64, t.data_ptr(), 8, 0.5, row.data_ptr(),
                                 None if which else out.data_ptr(), 64, out.data_ptr() if which else None, 64,
                                 ws.data_ptr(), ws.numel(), s.cuda_stream)
            assert rc == K.OK
            lm.sync()
            assert torch.equal(row, loss) and torch.equal(out, dw if which else dh)


@pytest.mark.gpu
def test_in_a_graph(lm):
    h, w, t = _case(200, 64, 500, "bf16")
    want = lm.xent(h, w, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = lm.xent(h, w, t)
    for x in got:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_wrapper_refuses(lm):
    h, w, t = torch.zeros(4, 16, device="cuda"), torch.zeros(9, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: lm.xent(h, w[:, :8], t), lambda: lm.xent(h, w.bfloat16(), t), lambda: lm.xent(h, w, t[:3]),
                 lambda: lm.xent(h, w, t.float()), lambda: lm.xent(h.double(), w.double(), t), lambda: lm.xent(h, w.cpu(), t),
                 lambda: lm.xent(h, w, t, grad=False, dh=h), lambda: lm.xent(h, w, t, dw=h), lambda: lm.xent(h.t(), w, t)):
        with pytest.raises(ValueError):
            call()


def test_c_entry_refuses_before_any_device_work(native):
    import ctypes as C
    from tbb_test_b200 import _capi as K
    lib, p = K.lib(), C.c_void_p(256)
    good = dict(rows=3, width=8, vocab=5, dtype=0, h=p, ldh=8, w=p, ldw=8, t=p, size=8, scale=1.0, loss=p, dh=p, lddh=8, dw=p,
                lddw=8, ws=p, ws_bytes=1 << 30, stream=None)

    def xent(**kw):
        return lib.b2_xent(*{**good, **kw}.values())

    for kw in (dict(rows=(1 << 24) + 1), dict(width=0), dict(width=(1 << 20) + 1), dict(vocab=0), dict(vocab=1 << 25), dict(rows=1 << 23, vocab=1 << 22), dict(dtype=3),
               dict(h=None), dict(w=None), dict(t=None), dict(loss=None), dict(ws=None), dict(ldh=7), dict(ldw=7), dict(lddh=7),
               dict(lddw=7), dict(size=1), dict(ws=C.c_void_p(128)), dict(ws_bytes=100), dict(h=C.c_void_p(258)),
               dict(t=C.c_void_p(260)), dict(dw=C.c_void_p(257))):
        assert xent(**kw) == K.ERR_INVALID, kw
        assert lib.b2_last_error(None)
    need = C.c_size_t()
    assert lib.b2_xent_workspace(3, 8, 5, 0, 1, p, 8, C.byref(need)) == K.OK and need.value > 0
    assert lib.b2_xent_workspace(3, 8, 5, 0, 1, p, 8, None) == K.ERR_INVALID
    aligned, odd = C.c_size_t(), C.c_size_t()
    lib.b2_xent_workspace(300, 64, 5000, 1, 1, p, 64, C.byref(aligned))
    lib.b2_xent_workspace(300, 64, 5000, 1, 1, p, 65, C.byref(odd))
    assert odd.value >= aligned.value + 5000 * 64 * 2  # a copy of w, as its rows are no whole 16-byte pieces
