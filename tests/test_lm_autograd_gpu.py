"""What autograd sees of the operators: nothing of what they compute, everything that they write into given tensors."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lm(native):
    from tbb_test_b200 import lm
    return lm


def _calls(lm):
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = torch.randint(0, 30, (20,), device="cuda", generator=g)
    table, dout, h, w, m, grad = r(30, 16), r(20, 16), r(20, 16), r(30, 16), r(2, 30, 16), r(2, 30, 16)
    pair, copies = r(2, 30, 16), torch.zeros(2, 30, 16, device="cuda", dtype=torch.bfloat16)
    return [(r(20, 16), lambda x: lm.embed(t, table, out=x)), (r(30, 16), lambda x: lm.embed_grad(t, dout, 30, out=x)),
            (r(20, 16), lambda x: lm.xent(h, w, t, dh=x)), (r(30, 16), lambda x: lm.xent(h, w, t, dw=x)),
            (r(2, 30, 16), lambda x: lm.muon(x, m, grad, lr=0.1)), (r(2, 30, 16), lambda x: lm.muon(list(pair), x, grad, lr=0.1)),
            (r(30, 16), lambda x: lm.muon([pair[0], x], list(m), grad, lr=0.1)), (copies, lambda x: lm.muon(pair, m, grad, lr=0.1, copy=x))]


@pytest.mark.parametrize("which", range(8))
def test_a_saved_value_that_a_call_writes_over_is_refused(lm, which):
    x, call = _calls(lm)[which]
    x.requires_grad_()
    y = (x * x).sum()  # keeps x for its backward pass
    call(x.detach())  # shares x's count of changes
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    z = (x * x).sum()
    z.backward()
    assert torch.equal(x.grad, 2 * x.detach())


@pytest.mark.parametrize("which", range(8))
def test_under_inference_mode(lm, which):
    with torch.inference_mode():
        x, call = _calls(lm)[which]
        before = x.clone()
        call(x)
        assert not torch.equal(x, before)


def test_results_require_no_gradient(lm):
    t = torch.arange(20, device="cuda")
    h, w = (torch.randn(20, 16, device="cuda", requires_grad=True) for _ in range(2))
    for x in (lm.embed(t, w), lm.embed_grad(t, h, 20), *lm.xent(h, w, t)):
        assert not x.requires_grad
    assert h.grad is None and w.grad is None
    before = [x._version for x in (t, h, w)]
    lm.xent(h, w, t)
    assert [x._version for x in (t, h, w)] == before
