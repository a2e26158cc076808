"""Operators around the layers of a language model, on torch tensors of one GPU.

  embed, embed_grad   rows of a table by token number, and the table's gradient
  xent                softmax cross entropy behind a linear layer as wide as a vocabulary, with its gradients
  sync                waits for the current stream and raises if a kernel's bounded wait gave up

Thin wrappers over the C ABI (include/b200mlp.h, "Operators around the layers of a language model"): they
check shapes, types and devices, allocate what is returned, and queue the work on the current torch stream without waiting
for it. Matrices are float32 or bfloat16, all of one call alike, with unit stride along rows and any distance between
rows. Tokens are int32 or int64; one outside [0, vocab) is padding. There is no CPU path.
"""
import ctypes as C

import torch

from . import _capi as K

_DTYPES = {torch.float32: K.DTYPE_F32, torch.bfloat16: K.DTYPE_BF16}


def _ck(rc):
    if rc != K.OK:
        raise K.B2Error(rc, K.lib().b2_last_error(None).decode())


def _matrix(name, x, dtype=None, shape=None, device=None):
    """(address, leading dimension) of a two-dimensional CUDA tensor with unit stride along its rows."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{name}: a two-dimensional tensor is wanted")
    if not x.is_cuda or (device is not None and x.device != device):
        raise ValueError(f"{name}: on {x.device}, wanted on {device if device is not None else 'a CUDA device'}")
    if x.dtype not in _DTYPES or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{name}: {x.dtype}, wanted {dtype if dtype is not None else 'float32 or bfloat16'}")
    if shape is not None and tuple(x.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, wanted {tuple(shape)}")
    if x.shape[1] > 1 and x.stride(1) != 1:
        raise ValueError(f"{name}: rows need unit stride")
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        raise ValueError(f"{name}: rows overlap")
    return x.data_ptr(), max(x.stride(0), x.shape[1]) if x.shape[0] > 1 else x.shape[1]


def _tokens(name, t, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: an int32 or int64 tensor is wanted")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, wanted on {device}")
    t = t.reshape(-1).contiguous()
    return t, t.element_size()


def _workspace(size, device):
    """Device memory from torch's allocator, which hands it out again only behind this stream's work."""
    return torch.empty(max(int(size), 1), dtype=torch.uint8, device=device)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def embed(tokens, table, scale=1.0, out=None):
    """`scale * table[tokens]`: one row per token in the order of `tokens.reshape(-1)`; zeros for padding."""
    p, ld = _matrix("table", table)
    vocab, width = table.shape
    t, size = _tokens("tokens", tokens, table.device)
    n = t.numel()
    if out is None:
        out = torch.empty(n, width, dtype=table.dtype, device=table.device)
    po, ldo = _matrix("out", out, table.dtype, (n, width), table.device)
    with torch.cuda.device(table.device):
        _ck(K.lib().b2_embed(t.data_ptr(), size, n, p, _DTYPES[table.dtype], vocab, width, ld, scale, po, ldo,
                             _stream(table.device)))
    return out


def embed_grad(tokens, dout, vocab, scale=1.0, out=None):
    """Gradient of `embed` with respect to the table, vocab x width, from the gradient `dout` of its output."""
    p, ld = _matrix("dout", dout)
    n, width = dout.shape
    t, size = _tokens("tokens", tokens, dout.device)
    if t.numel() != n:
        raise ValueError(f"dout: {n} rows for {t.numel()} tokens")
    if out is None:
        out = torch.empty(vocab, width, dtype=dout.dtype, device=dout.device)
    po, ldo = _matrix("out", out, dout.dtype, (vocab, width), dout.device)
    need = C.c_size_t()
    _ck(K.lib().b2_embed_grad_workspace(n, vocab, width, C.byref(need)))
    with torch.cuda.device(dout.device):
        ws = _workspace(need.value, dout.device)
        _ck(K.lib().b2_embed_grad(t.data_ptr(), size, n, p, _DTYPES[dout.dtype], ld, vocab, width, scale, po, ldo,
                                  ws.data_ptr(), ws.numel(), _stream(dout.device)))
    return out


def xent(h, w, targets, scale=1.0, grad=True, dh=None, dw=None):
    """Losses of `h @ w.T` against `targets`, one float32 per row (0 for padding); with `grad` also the gradients of
    `scale * losses.sum()` with respect to h and w: (losses, dh, dw). `dh` and `dw` may be given to be written to. The logits
    are never kept (see b2_xent in include/b200mlp.h)."""
    ph, ldh = _matrix("h", h)
    rows, width = h.shape
    device, dtype = h.device, h.dtype
    pw, ldw = _matrix("w", w, dtype, (w.shape[0], width) if w.dim() == 2 else None, device)
    vocab = w.shape[0]
    t, size = _tokens("targets", targets, device)
    if t.numel() != rows:
        raise ValueError(f"targets: {t.numel()} for {rows} rows")
    if not grad and (dh is not None or dw is not None):
        raise ValueError("dh and dw go with grad=True")
    loss = torch.empty(rows, dtype=torch.float32, device=device)
    pdh = pdw = None
    lddh = lddw = 0
    if grad:
        dh = torch.empty(rows, width, dtype=dtype, device=device) if dh is None else dh
        dw = torch.empty(vocab, width, dtype=dtype, device=device) if dw is None else dw
        pdh, lddh = _matrix("dh", dh, dtype, (rows, width), device)
        pdw, lddw = _matrix("dw", dw, dtype, (vocab, width), device)
    need = C.c_size_t()
    _ck(K.lib().b2_xent_workspace(rows, width, vocab, _DTYPES[dtype], int(grad), pw, ldw, C.byref(need)))
    with torch.cuda.device(device):
        ws = _workspace(need.value, device)
        _ck(K.lib().b2_xent(rows, width, vocab, _DTYPES[dtype], ph, ldh, pw, ldw, t.data_ptr(), size, scale,
                            loss.data_ptr(), pdh, lddh, pdw, lddw, ws.data_ptr(), ws.numel(), _stream(device)))
    return (loss, dh, dw) if grad else loss


def sync(device=None):
    """Waits for the current stream of `device`; K.B2Error with code ERR_TIMEOUT if a bounded wait of a kernel gave up."""
    device = torch.device("cuda" if device is None else device)
    with torch.cuda.device(device):
        _ck(K.lib().b2_lm_sync(_stream(device)))
