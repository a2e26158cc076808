"""Norm, clipping and sampling as they are used together, and what holds for every operator: workspaces whose contents do not matter, autograd's count of changes,
streams side by side, offsets beyond 32 bits."""
import ctypes as ct
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


@pytest.fixture(scope="module")
def example(native):
    from tbb_test_b200 import lm_example
    return lm_example


def _exact_loss(model, contexts, targets):
    table, c, w, gain = (t.double().requires_grad_() for t in (model.table, model.c, model.w, model.gain))
    rows = torch.where((contexts >= 0)[..., None], table[contexts.clamp(min=0)], 0.0).reshape(len(contexts), -1)
    t = rows @ c.T
    h = t / torch.sqrt(t.square().mean(1, keepdim=True) + float(torch.tensor(1e-6))) * gain
    x = h @ w.T
    ok = targets >= 0
    loss = torch.where(ok, torch.logsumexp(x, 1) - x.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    return loss, x, (table, c, w, gain)


def test_one_step_of_a_model_with_all_of_them(example, lm):
    """Gradients with a norm between the layers against torch in 64 bits. All products are fp32-class and sums have at most 700 terms, 500 for the gain's gradient: 2^-24 *
    700 of the magnitudes is 4e-5 at worst, and rounding errors of such sums are far apart in sign: 1e-5 of each gradient's norm."""
    model = example.LogBilinear(vocab=700, width=24, hidden=40, context=3, seed=4, norm=True)
    contexts, targets = next(example.batches(example.synthetic_text(5000, 700, 1), 3, 500, 2))
    contexts[0] = -1
    targets[5:9] = -1
    model.gain.uniform_(0.5, 1.5, generator=torch.Generator(device="cuda").manual_seed(1))
    loss, *grads = model.gradients(contexts, targets)
    want, _, leaves = _exact_loss(model, contexts, targets)
    (want.sum() / 500).backward()
    want = want.detach()
    assert float((loss.double() - want).abs().max()) <= 1e-5 * float(want.max())
    for got, leaf in zip(grads, leaves):
        assert float(torch.linalg.norm(got.double() - leaf.grad)) <= 1e-5 * float(torch.linalg.norm(leaf.grad))
    # clipped, all together
    total = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    before = [g.clone() for g in grads]
    norm = lm.clip(grads, 0.25 * total)
    assert abs(float(norm) - total) <= 1e-6 * total
    for g, b in zip(grads, before):
        assert float((g - 0.25 * b).abs().max()) <= 1e-6 * float(b.abs().max())
    first = model.step(contexts, targets, max_norm=0.25 * total)
    assert abs(float(first) - float(want.mean())) <= 1e-5 * float(want.mean())
    lm.sync()
    model.close()


def test_continuing_a_text(example, lm):
    """The tokens of the model's own logits: greedy ones are the most probable, and the others those of the running sum in 64 bits."""
    model = example.LogBilinear(vocab=300, width=16, hidden=32, context=3, seed=2, norm=True)
    start = example.synthetic_text(30, 300, 5).view(10, 3)
    u = torch.rand(6, 10, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    greedy = model.generate(start, u, temperature=0.0)
    tokens = model.generate(start, u, temperature=0.75)
    assert greedy.shape == tokens.shape == (10, 6)
    text, text2 = torch.cat([start, greedy], 1), torch.cat([start, tokens], 1)
    for i in range(6):
        x = model._sgemm(model.forward(text[:, i:i + 3].contiguous())[2], model.w, False, True)
        assert torch.equal(x.argmax(1), greedy[:, i])
        x = model._sgemm(model.forward(text2[:, i:i + 3].contiguous())[2], model.w, False, True)
        p = torch.softmax(x.double() / 0.75, 1).cumsum(1)
        assert torch.equal((p <= u[i].double()[:, None] * p[:, -1:]).sum(1), tokens[:, i])
    model.close()


def test_example_runs(example, monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["lm_example", "--steps", "3", "--batch", "256", "--norm", "--clip", "1", "--generate", "4"])
    example.main()
    assert "|" in capsys.readouterr().out


def _writes(lm):
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, res, w, u = r(20, 16), r(20, 16), r(16), torch.rand(20, device="cuda", generator=g)
    return [(r(20, 16), lambda t: lm.norm(x, w, out=t)), (r(20, 16), lambda t: lm.norm(x, w, res, total=t)), (r(20, 16), lambda t: lm.norm_e4m3(x, w, res, total=t)),
            (r(20, 16), lambda t: lm.norm_grad(x, res, w, dx=t)), (r(20, 16), lambda t: lm.clip([x, t], 0.1)), (r(20, 16), lambda t: lm.clip([x], 0.1, out=[t])),
            (r(20, 16), lambda t: lm.sample(x, u, out=t.view(-1).view(torch.int32)[:20]))]


@pytest.mark.parametrize("which", range(7))
def test_a_saved_value_that_a_call_writes_over_is_refused(lm, which):
    t, call = _writes(lm)[which]
    t.requires_grad_()
    y = (t * t).sum()
    call(t.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("which", range(7))
def test_under_inference_mode(lm, which):
    with torch.inference_mode():
        t, call = _writes(lm)[which]
        before = t.clone()
        call(t)
        assert not torch.equal(t, before)


def test_results_require_no_gradient(lm):
    x, w = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((8, 16), (16,)))
    q, s, t = lm.norm_e4m3(x, w, x)
    for y in (*lm.norm(x, w, x), q, s, t, *lm.norm_grad(x, x, w), lm.clip([x.detach().clone()], 1.0), *lm.sample(x, torch.rand(8, device="cuda"), logprob=True)):
        assert not y.requires_grad


def test_what_a_workspace_holds_does_not_matter(lm):
    """The C ABI with workspaces of every byte 0xFF, 0 and 0x7F, of exactly the size that is asked for."""
    from tbb_test_b200 import _capi as K
    lib = K.lib()
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    dy, t, w, x = r(700, 520), r(700, 520), r(520), r(30, 40000) * 2.5
    u = torch.rand(30, device="cuda", generator=g)
    xs = [r(5000 + i) for i in range(50)]
    want = lm.norm_grad(dy, t, w), lm.clip(xs, None), [lm.sample(x, u, logprob=True, **o) for o in (dict(), dict(top_p=0.9), dict(top_k=30))]
    need = ct.c_size_t()
    for fill in (0xFF, 0, 0x7F):
        def space(entry, *sizes):
            assert getattr(lib, f"b2_{entry}_workspace")(*sizes, ct.byref(need)) == K.OK
            buf = torch.full((need.value + 4096,), fill, dtype=torch.uint8, device="cuda")
            return buf, buf.data_ptr(), need.value
        dx, dw = torch.empty_like(dy), torch.empty_like(w)
        buf, p, n = space("norm_grad", 700, 520, 0)
        assert lib.b2_norm_grad(700, 520, 0, dy.data_ptr(), 520, t.data_ptr(), 520, None, 0, w.data_ptr(), 0, 1e-6, dx.data_ptr(), 520, dw.data_ptr(), p, n, None) == K.OK
        torch.cuda.synchronize()
        assert torch.equal(dx, want[0][0]) and torch.equal(dw, want[0][1]) and bool((buf[n:] == fill).all())
        buf, p, n = space("clip", 50)
        norm = torch.empty((), device="cuda")
        ptrs, sizes, types = (ct.c_void_p * 50)(*[v.data_ptr() for v in xs]), (ct.c_size_t * 50)(*[v.numel() for v in xs]), (ct.c_int * 50)()
        assert lib.b2_clip(50, ptrs, None, sizes, types, None, None, None, math.inf, norm.data_ptr(), p, n, None) == K.OK
        torch.cuda.synchronize()
        assert torch.equal(norm, want[1]) and bool((buf[n:] == fill).all())
        for o, (tokens, lp) in zip((dict(), dict(top_p=0.9), dict(top_k=30)), want[2]):
            buf, p, n = space("sample", 30, 40000)
            got, glp, opt = torch.empty_like(tokens), torch.empty_like(lp), K.SampleOptions()
            assert lib.b2_sample_options_default(ct.byref(opt)) == K.OK
            for k, v in o.items():
                setattr(opt, k, v)
            assert lib.b2_sample(30, 40000, 0, x.data_ptr(), 40000, u.data_ptr(), ct.byref(opt), got.data_ptr(), 8, glp.data_ptr(), p, n, None) == K.OK
            torch.cuda.synchronize()
            assert torch.equal(got, tokens) and torch.equal(glp, lp) and bool((buf[n:] == fill).all())


def test_calls_on_two_streams_side_by_side(lm):
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    data = [(r(3000, 1024).bfloat16(), r(1024), r(64, 50000) * 2, torch.rand(64, device="cuda", generator=g), [r(1 << 20), r(12345)]) for _ in range(2)]

    def calls(x, w, logits, u, xs):
        y, t = lm.norm(x, w, x)
        return [y, t, *lm.norm_grad(y, t, w), lm.clip(xs, 1.0, out=[torch.empty_like(v) for v in xs]), lm.sample(logits, u, top_p=0.8), lm.sample(logits, u), lm.sample(logits, u, top_k=9)]

    want = [calls(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(calls(*data[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(one, want[i]))


def test_two_graphs_in_turn(lm):
    """Each graph has workspaces of its own; replayed in turn and one behind the other they give what the calls gave."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x = [torch.randn(40, 30000, device="cuda", generator=g) * 2 for _ in range(2)]
    u = torch.rand(40, device="cuda", generator=g)
    want = [lm.sample(v, u, top_p=0.9) for v in x] + [lm.sample(v, u) for v in x]
    graphs, got = [], []
    for f in (lambda v: lm.sample(v, u, top_p=0.9), lambda v: lm.sample(v, u)):
        for v in x:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got.append(f(v))
            graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_offsets_beyond_32_bits(lm):
    """Rows that lie 2^32 bytes apart, and one tensor of more than 2^31 elements."""
    far = (1 << 31) + 64  # bf16 elements
    buf = torch.zeros(2 * far, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    rows = torch.randn(2, 4096, device="cuda", generator=g).bfloat16()
    x = buf.as_strided((2, 4096), (far, 1))
    x.copy_(rows)
    u = torch.tensor([0.3, 0.9], device="cuda")
    assert torch.equal(lm.norm(x), lm.norm(rows))
    assert torch.equal(lm.norm_grad(x, x), lm.norm_grad(rows, rows))
    for o in (dict(), dict(top_k=20), dict(top_p=0.7)):
        assert torch.equal(lm.sample(x, u, **o), lm.sample(rows, u, **o))
    whole = rows.double().square().sum().sqrt()
    assert abs(float(lm.clip([buf], 1.0)) - float(whole)) <= 5 * 2.0 ** -24 * float(whole)
    exact = rows.double() / whole
    assert bool(((x.double() - exact).abs() <= exact.abs() * (6 * 2.0 ** -24 + 2.0 ** -8)).all())
