"""Training of a log-bilinear language model with this package's operators, on one GPU.

The next token's logits are a linear function of the embeddings of the `context` tokens before it:

    x_i = [E[t_{i-context}] ... E[t_{i-1}]]        lm.embed
    h_i = x_i C'                                   b2_sgemm
    loss = mean of -log softmax(h_i W')[t_i]       lm.xent, with the gradients of h and W

and backwards: dC = dh' x and dx = dh C (b2_sgemm), dE by lm.embed_grad. The hidden matrix C is updated by lm.muon, the
embeddings and W by plain gradient steps.

    python -m tbb_test_b200.lm_example --steps 100

The text is synthetic: each token follows from the one before it three times out of four and is drawn at random otherwise, which a
model of this kind can learn: the best possible loss is well below that of guessing.
"""
import argparse

import torch

from . import _capi as K
from . import lm
from .mlp import MLP


def synthetic_text(length, vocab, seed, device="cuda"):
    """`length` tokens; a token is a fixed function of the one before it, or with probability 1/4 any other."""
    g = torch.Generator().manual_seed(seed)
    noise = torch.randint(0, vocab, (length,), generator=g).tolist()
    free = (torch.rand(length, generator=g) < 0.25).tolist()
    text = noise[:1]
    for i in range(1, length):
        text.append(noise[i] if free[i] else (7 * text[-1] + 1) % vocab)
    return torch.tensor(text, device=device)


class LogBilinear:
    def __init__(self, vocab, width, hidden, context, seed=0, device="cuda"):
        self.vocab, self.width, self.hidden, self.context = vocab, width, hidden, context
        g = torch.Generator(device=device).manual_seed(seed)
        randn = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
        self.table = randn(vocab, width) * width ** -0.5
        self.c = randn(hidden, context * width) * (context * width) ** -0.5
        self.w = randn(vocab, hidden) * hidden ** -0.5
        self.momentum = torch.zeros_like(self.c)
        self.gemms = MLP([8, 8], 8, device=self.table.device.index)  # the handle whose stream b2_sgemm runs on

    def _sgemm(self, a, b, transa, transb):
        """op(a) op(b) in fp32. The handle has a stream of its own: torch's is waited for before, and it after."""
        m, k = a.shape[::-1] if transa else a.shape
        n = b.shape[0] if transb else b.shape[1]
        out = torch.empty(m, n, device=a.device)
        torch.cuda.current_stream(a.device).synchronize()
        rc = K.lib().b2_sgemm(self.gemms._h, K.PREC_FP32, int(transa), int(transb), m, n, k, 1.0, a.data_ptr(), a.shape[1], b.data_ptr(),
                              b.shape[1], 0.0, out.data_ptr(), n)
        self.gemms._ck(rc)
        self.gemms.sync()
        return out

    def gradients(self, contexts, targets):
        """Per-position losses and the gradients of their mean. contexts: positions x context tokens; padding is allowed."""
        n = targets.numel()
        x = lm.embed(contexts, self.table).view(n, self.context * self.width)
        h = self._sgemm(x, self.c, False, True)
        loss, dh, dw = lm.xent(h, self.w, targets, scale=1.0 / n)
        dc = self._sgemm(dh, x, True, False)
        dx = self._sgemm(dh, self.c, False, False)
        dtable = lm.embed_grad(contexts, dx.view(n * self.context, self.width), self.vocab)
        return loss, dtable, dc, dw

    def step(self, contexts, targets, lr=0.5, lr_hidden=0.02):
        """One update; the mean loss before it, on the device."""
        loss, dtable, dc, dw = self.gradients(contexts, targets)
        self.table.add_(dtable, alpha=-lr * self.vocab ** 0.5)
        self.w.add_(dw, alpha=-lr * self.vocab ** 0.5)
        lm.muon([self.c], [self.momentum], [dc], lr=lr_hidden, momentum=0.9)
        return loss.mean()

    def close(self):
        self.gemms.close()


def batches(text, context, size, seed):
    """Endless (contexts, targets) at random positions; a context that would begin before the text is padded with -1."""
    g = torch.Generator().manual_seed(seed)
    padded = torch.cat([torch.full((context,), -1, device=text.device, dtype=text.dtype), text])
    window = padded.unfold(0, context + 1, 1)
    while True:
        rows = window[torch.randint(0, len(text), (size,), generator=g).to(text.device)]
        yield rows[:, :context].contiguous(), rows[:, context].contiguous()


def main():
    p = argparse.ArgumentParser(description="Trains a log-bilinear language model on synthetic text.")
    p.add_argument("--vocab", type=int, default=128)
    p.add_argument("--width", type=int, default=64)
    p.add_argument("--hidden", type=int, default=128)
    p.add_argument("--context", type=int, default=4)
    p.add_argument("--batch", type=int, default=4096)
    p.add_argument("--steps", type=int, default=200)
    a = p.parse_args()
    model = LogBilinear(a.vocab, a.width, a.hidden, a.context)
    stream = batches(synthetic_text(1 << 17, a.vocab, 1), a.context, a.batch, 2)
    for i in range(a.steps):
        loss = model.step(*next(stream))
        if i % 20 == 0 or i == a.steps - 1:
            print(f"step {i:4d}  loss {float(loss):.4f}")
    lm.sync()
    model.close()


if __name__ == "__main__":
    main()
