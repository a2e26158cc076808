"""The operators together, as the example runs them: one training step against torch in 64 bits, and a loss that falls."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def example(native):
    from tbb_test_b200 import lm_example
    return lm_example


@pytest.mark.gpu
def test_gradients_of_the_whole_model(example):
    """All products are fp32-class and sums have at most 700 terms: 2^-24 * 700 of the magnitudes is 4e-5 at worst, and
    rounding errors of such sums are far apart in sign: 1e-5 of each gradient's norm."""
    model = example.LogBilinear(vocab=700, width=24, hidden=40, context=3, seed=4)
    contexts, targets = next(example.batches(example.synthetic_text(5000, 700, 1), 3, 500, 2))
    contexts[0] = -1
    targets[5:9] = -1  # no loss, no gradient
    loss, dtable, dc, dw = model.gradients(contexts, targets)
    table, c, w = (t.double().requires_grad_() for t in (model.table, model.c, model.w))
    rows = torch.where((contexts >= 0)[..., None], table[contexts.clamp(min=0)], 0.0).reshape(500, -1)
    x = rows @ c.T @ w.T
    ok = targets >= 0
    want = torch.where(ok, torch.logsumexp(x, 1) - x.gather(1, targets.clamp(min=0)[:, None])[:, 0], 0.0)
    (want.sum() / 500).backward()
    want = want.detach()
    assert float((loss.double() - want).abs().max()) <= 1e-5 * float(want.max())
    for got, exact in ((dtable, table.grad), (dc, c.grad), (dw, w.grad)):
        assert float(torch.linalg.norm(got.double() - exact)) <= 1e-5 * float(torch.linalg.norm(exact))
    model.close()


@pytest.mark.gpu
def test_training_learns(example):
    """Guessing among 64 tokens costs log 64 = 4.16; the text is three quarters predictable."""
    model = example.LogBilinear(vocab=64, width=32, hidden=64, context=4)
    stream = example.batches(example.synthetic_text(1 << 15, 64, 1), 4, 1024, 2)
    losses = [float(model.step(*next(stream))) for _ in range(150)]
    assert 3.9 < losses[0] < 5.5
    assert sum(losses[-10:]) / 10 < losses[0] - 0.5
    model.close()


def test_synthetic_text_and_batches(example):
    text = example.synthetic_text(4000, 50, 3, device="cpu")
    follows = (7 * text[:-1] + 1) % 50 == text[1:]
    assert 0.7 < float(follows.double().mean()) < 0.82 and int(text.max()) < 50
    contexts, targets = next(example.batches(text, 3, 100, 0))
    assert contexts.shape == (100, 3) and targets.shape == (100,)
