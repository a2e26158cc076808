"""Arguments of the operators that share memory: refused where one of them is written, and only then."""
import ctypes as C
import random

import pytest

torch = pytest.importorskip("torch")


def test_the_rule(native):
    """Against a list of every byte: rows with gaps, in one another's gaps, at the same distance and at others, single rows, nothing."""
    host = C.CDLL(native.HOST_LIB)
    rng = random.Random(5)
    seen = {True: 0, False: 0}
    for trial in range(20000):
        n = rng.choice([2, 2, 3, 5])
        same = rng.randint(1, 24)
        x = []
        for _ in range(n):
            ld = same if rng.random() < 0.7 else rng.randint(1, 24)
            x.append((256 + rng.randint(0, 150), rng.choice([0, 1, 1, 2, 3, 8]), rng.randint(0 if rng.random() < 0.1 else 1, max(1, ld // 2)), ld, rng.random() < 0.5))
        at, rows, row, ld, written = zip(*x)
        out = (C.c_int * 2)()
        size = C.c_size_t * n
        got = host.b2h_any_overlap(n, size(*at), size(*rows), size(*row), size(*ld), (C.c_int * n)(*written), out)
        bytes_ = [{a + r * d + b for r in range(k) for b in range(c)} for a, k, c, d, _ in x]
        want = any((written[i] or written[j]) and bytes_[i] & bytes_[j] for i in range(n) for j in range(i))
        assert bool(got) == want, x
        if got:
            i, j = out
            assert (written[i] or written[j]) and bytes_[i] & bytes_[j]
        seen[want] += 1
    assert min(seen.values()) > 3000


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


@pytest.mark.gpu
def test_calls_that_overlap_are_refused(lm):
    from tbb_test_b200._capi import ERR_INVALID, B2Error
    buf = torch.randn(64, 64, device="cuda")
    t = torch.zeros(16, dtype=torch.int64, device="cuda")
    h, w, rest = buf[:16], buf[16:40], buf[40:]
    x = torch.randn(4, 16, 32, device="cuda")
    a, b, c = x[:1], x[1:2], x[2:3]
    before = buf.clone(), x.clone()
    for call in (lambda: lm.embed(t, buf, out=buf[:16]), lambda: lm.embed(t, buf[:24], out=buf[23:39]), lambda: lm.embed_grad(t, buf[:16], 24, out=buf[:24]),
                 lambda: lm.xent(h, w, t, dw=w), lambda: lm.xent(h, w, t, dh=h), lambda: lm.xent(h, w, t, dh=w[:16]), lambda: lm.xent(h, w, t, dw=buf[39:63]),
                 lambda: lm.xent(h, w, t, dh=rest[:16], dw=rest[:24]), lambda: lm.muon(a, a, c, lr=1.0), lambda: lm.muon(a, b, a, lr=1.0),
                 lambda: lm.muon([x[0], x[0]], [x[1], x[2]], [x[3], x[3]], lr=1.0), lambda: lm.muon([x[0]], [x[1]], [x[2]], lr=1.0, copy=[x[0, :8].view(torch.bfloat16).view(16, 32)])):
        with pytest.raises(B2Error) as e:
            call()
        assert e.value.code == ERR_INVALID and "overlap" in str(e.value)
    torch.cuda.synchronize()
    assert torch.equal(buf, before[0]) and torch.equal(x, before[1])


@pytest.mark.gpu
def test_matrices_side_by_side_are_not(lm):
    """Columns of one buffer, one gradient for two matrices, many matrices whose rows alternate."""
    g = torch.Generator(device="cuda").manual_seed(1)
    buf = torch.randn(40, 200, device="cuda", generator=g)
    t = torch.randint(0, 24, (16,), device="cuda", generator=g)
    want = lm.xent(buf[:16, :64].clone(), buf[16:40, :64].clone(), t)
    got = lm.xent(buf[:16, :64], buf[16:40, :64], t, dh=buf[:16, 64:128], dw=buf[16:40, 128:192])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.equal(lm.embed(t, buf[:24, :64], out=buf[3:19, 64:128]), buf[t, :64])
    for count in (3, 40):
        x = torch.randn(24, 2 * count, 32, device="cuda", generator=g)
        every = list(x.unbind(1))
        w, m, grad = every[:count], every[count:], torch.randn(24, 32, device="cuda", generator=g)
        w2, m2 = [p.clone() for p in w], [p.clone() for p in m]
        lm.muon(w2, m2, [grad] * count, lr=0.1)
        lm.muon(w, m, [grad] * count, lr=0.1)
        assert all(torch.equal(p, q) for p, q in zip(w + m, w2 + m2))
    lm.sync()
