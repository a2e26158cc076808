"""Operators around the layers of a language model, on torch tensors of one GPU.

  embed, embed_grad   rows of a table by token number, and the table's gradient
  xent                softmax cross entropy behind a linear layer as wide as a vocabulary, with its gradients
  norm, norm_e4m3     root-mean-square norm with the residual stream's addition, also with an output in 8 bits with scales
  norm_grad           its gradients
  clip                global norm of a list of gradients, and the gradients scaled down to a limit
  muon                momentum and an orthogonalised update of weight matrices
  sample              a token per row of logits: temperature, top-k, top-p, min-p
  sync                waits for the current stream and raises if a kernel's bounded wait gave up

Thin wrappers over the C ABI (include/b200mlp.h, "Operators around the layers of a language model"), those of norm, clip and sample in C++ (native/lm_native.cc): they
check shapes, types and devices (and the entries behind them overlaps), allocate what is returned, and queue the work on the current torch stream without waiting
for it. Matrices are float32 or bfloat16, all of one call alike, with unit stride along rows and any distance between
rows. Tokens are int32 or int64; one outside [0, vocab) is padding. There is no CPU path.

Nothing here is recorded by autograd, whatever its arguments require: results require no gradient, and embed_grad, norm_grad and xent give
the gradients themselves. What a call writes into a given tensor counts as an in-place change, so that autograd's own backward passes refuse
to use a value that it saved before.
"""
import ctypes as C
import functools

import torch

from . import _capi as K

_DTYPES = {torch.float32: K.DTYPE_F32, torch.bfloat16: K.DTYPE_BF16}


def _ck(rc):
    if rc != K.OK:
        raise K.B2Error(rc, K.lib().b2_last_error(None).decode())


def _matrix(name, x, dtype=None, shape=None, device=None):
    """(address, leading dimension) of a two-dimensional CUDA tensor with unit stride along its rows."""
    if isinstance(x, torch.Tensor) and x.dim() == 2 and x.is_contiguous() and (x.is_cuda if device is None else x.device == device) and (
            x.dtype in _DTYPES and dtype in (None, x.dtype)) and (shape is None or x.shape == shape):
        return x.data_ptr(), x.shape[1]  # what most callers give
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{name}: a two-dimensional tensor is wanted")
    if not x.is_cuda or (device is not None and x.device != device):
        raise ValueError(f"{name}: on {x.device}, wanted on {device if device is not None else 'a CUDA device'}")
    if x.dtype not in _DTYPES or (dtype is not None and x.dtype != dtype):
        raise ValueError(f"{name}: {x.dtype}, wanted {dtype if dtype is not None else 'float32 or bfloat16'}")
    rows, cols = x.shape
    if shape is not None and (rows, cols) != tuple(shape):
        raise ValueError(f"{name}: shape {(rows, cols)}, wanted {tuple(shape)}")
    between, along = x.stride()
    if cols > 1 and along != 1:
        raise ValueError(f"{name}: rows need unit stride")
    if rows <= 1:
        between = cols
    elif between < cols:
        raise ValueError(f"{name}: rows overlap")
    return x.data_ptr(), between


def _result(name, x, rows, cols, dtype, device, like=None):
    """(tensor, address, leading dimension) of a result: the given one, checked, or a new one. like: a matrix of its shape and type, if there is one."""
    if x is None:
        x = _new(device, dtype, rows, cols) if like is None or not like.is_contiguous() else torch.empty_like(like)
        return x, x.data_ptr(), cols
    return (x, *_matrix(name, x, dtype, (rows, cols), device))


@functools.lru_cache(maxsize=256)
def _template(device, dtype):
    """A tensor without elements: new ones made from it take half the time of torch.empty's with a type and a device."""
    return torch.empty(0, dtype=dtype, device=device)


def _new(device, dtype, *shape):
    return _template(device, dtype).new_empty(shape)


def _tokens(name, t, device):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: an int32 or int64 tensor is wanted")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, wanted on {device}")
    if t.dim() != 1 or not t.is_contiguous():
        t = t.reshape(-1).contiguous()
    return t, 8 if t.dtype == torch.int64 else 4


@functools.lru_cache(maxsize=256)
def _workspace_bytes(entry, *sizes):
    """What b2_<entry>_workspace says for these sizes."""
    need = C.c_size_t()
    _ck(getattr(K.lib(), f"b2_{entry}_workspace")(*sizes, C.byref(need)))
    return max(need.value, 1)


def _workspace(device, entry, *sizes):
    """Device memory from torch's allocator, which hands it out again only behind this stream's work."""
    return _new(device, torch.uint8, _workspace_bytes(entry, *sizes))


def _changed(tensors):
    """Given tensors that a call has written to: counted as changed in place where autograd keeps count."""
    try:
        torch.autograd.graph.increment_version(tensors)
    except RuntimeError:  # some were made in inference mode, which keeps no count; counting the others twice does no harm
        torch.autograd.graph.increment_version([x for x in tensors if not x.is_inference()])


class _on:
    """The device of a call made the current one, where it is not already; gives the address of its current stream."""

    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.index != self.before:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *a):
        if self.index != self.before:
            torch.cuda.set_device(self.before)


def embed(tokens, table, scale=1.0, out=None):
    """`scale * table[tokens]`: one row per token in the order of `tokens.reshape(-1)`; zeros for padding."""
    p, ld = _matrix("table", table)
    vocab, width = table.shape
    device = table.device
    t, size = _tokens("tokens", tokens, device)
    n = t.numel()
    given = [] if out is None else [out]
    out, po, ldo = _result("out", out, n, width, table.dtype, device)
    with _on(device) as stream:
        _ck(K.lib().b2_embed(t.data_ptr(), size, n, p, _DTYPES[table.dtype], vocab, width, ld, scale, po, ldo, stream))
    if given:
        _changed(given)
    return out


def embed_grad(tokens, dout, vocab, scale=1.0, out=None):
    """Gradient of `embed` with respect to the table, vocab x width, from the gradient `dout` of its output."""
    p, ld = _matrix("dout", dout)
    n, width = dout.shape
    device = dout.device
    t, size = _tokens("tokens", tokens, device)
    if t.numel() != n:
        raise ValueError(f"dout: {n} rows for {t.numel()} tokens")
    given = [] if out is None else [out]
    out, po, ldo = _result("out", out, vocab, width, dout.dtype, device)
    with _on(device) as stream:
        ws = _workspace(device, "embed_grad", n, vocab, width)
        _ck(K.lib().b2_embed_grad(t.data_ptr(), size, n, p, _DTYPES[dout.dtype], ld, vocab, width, scale, po, ldo,
                                  ws.data_ptr(), ws.numel(), stream))
    if given:
        _changed(given)
    return out


def xent(h, w, targets, scale=1.0, grad=True, dh=None, dw=None):
    """Losses of `h @ w.T` against `targets`, one float32 per row (0 for padding); with `grad` also the gradients of
    `scale * losses.sum()` with respect to h and w: (losses, dh, dw). `dh` and `dw` may be given to be written to. The
    workspace holds up to 512 MB of logits and 640 MB of their gradients beside copies of h and, in fp32, of w (see b2_xent in
    include/b200mlp.h)."""
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
    given = [x for x in (dh, dw) if x is not None]
    loss = torch.empty(rows, dtype=torch.float32, device=device)
    pdh = pdw = None
    lddh = lddw = 0
    if grad:
        dh, pdh, lddh = _result("dh", dh, rows, width, dtype, device, h)
        dw, pdw, lddw = _result("dw", dw, vocab, width, dtype, device, w)
    with _on(device) as stream:
        # the size goes by the alignment of w and its rows
        ws = _workspace(device, "xent", rows, width, vocab, _DTYPES[dtype], int(grad), pw % 256 or None, ldw)
        _ck(K.lib().b2_xent(rows, width, vocab, _DTYPES[dtype], ph, ldh, pw, ldw, t.data_ptr(), size, scale,
                            loss.data_ptr(), pdh, lddh, pdw, lddw, ws.data_ptr(), ws.numel(), stream))
    if given:
        _changed(given)
    return (loss, dh, dw) if grad else loss


@functools.lru_cache(maxsize=None)
def _native():
    """The C++ side of the calls below, with the entries of the library that this process uses."""
    try:
        from .native import _lm_native
    except ImportError as e:
        raise ImportError(f"{e}: build it with `python -m tbb_test_b200.build` (there is no CPU or PyTorch fallback)") from None
    entries = ("b2_norm", "b2_norm_grad_workspace", "b2_norm_grad", "b2_clip_workspace", "b2_clip", "b2_sample_workspace", "b2_sample", "b2_last_error")
    _lm_native.use(*[C.cast(getattr(K.lib(), name), C.c_void_p).value for name in entries], K.B2Error)
    return _lm_native


def norm(x, weight=None, residual=None, eps=1e-6, total=None, out=None):
    """`t / sqrt(mean of t's squares + eps) * weight` for each row of t = x, or of t = x + residual rounded to their type: then
    (norm, t), t to be added to by what comes next and for `norm_grad`. weight: one element per column, of the matrices' type or
    float32. `total` (t) and `out` may be given to be written to."""
    return _native().norm(x, weight, residual, eps, total, out, False, 0)


def norm_e4m3(x, weight=None, residual=None, eps=1e-6, block=128, total=None):
    """The same with its result in 8 bits, to stand in front of a product of such operands: (q, scales), or (q, scales, t) with a
    residual. q is float8_e4m3fn, and q * scale the norm: a float32 scale for each `block` = 128 columns, or for each row
    (block = 0), rows x scales. Gradients are those of `norm` (norm_grad)."""
    return _native().norm(x, weight, residual, eps, total, None, True, block)


def norm_grad(dy, t, weight=None, dtotal=None, eps=1e-6, dx=None):
    """Gradients of `norm` from the gradient dy of its result, at t (x, or x + residual as norm gave it): dx for x and residual
    alike, or (dx, dweight) with a weight. `dtotal`: a gradient that arrives at t elsewhere, which dx includes."""
    return _native().norm_grad(dy, t, weight, dtotal, eps, dx)


def clip(tensors, max_norm, out=None):
    """The norm of all elements of `tensors` together, a float32 scalar on their device; where it is over `max_norm`, the tensors are multiplied
    by max_norm / norm, in place or into the list `out` of tensors like them (which is always written). math.inf or None for max_norm: the
    norm alone. A norm that is infinite (in float32) or not a number leaves the values as they are. float32 and bfloat16 tensors of any sizes, each dense
    or a matrix with unit stride along its rows, all on one device; none may overlap another (see b2_clip in include/b200mlp.h)."""
    return _native().clip(tensors, max_norm, out)


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, logprob=False, out=None):
    """One token per row of `logits`, int64, by the uniform random numbers `u` (float32, one per row, from [0, 1)); with `logprob`
    also the logarithm of its probability among the tokens that were kept, float32: (tokens, logprobs).

    Kept are the top_k most probable tokens, of these the fewest whose probability reaches top_p, and of these the ones of at least
    min_p times the largest probability; tokens of one logit count in the order of their numbers. Each of the four may be a tensor with one
    for each row (float32; top_k int32). temperature 0 takes the most probable token. A logit of -inf or NaN is never taken; a row of nothing
    else gives -1. `out`, int64 or int32, may be given to be written to. See b2_sample in include/b200mlp.h."""
    return _native().sample(logits, u, temperature, top_k, top_p, min_p, logprob, out)


def _listed(x):
    """The matrices of a three-dimensional tensor, or of a sequence of them."""
    return list(x.unbind(0)) if isinstance(x, torch.Tensor) and x.dim() == 3 else list(x)


def _matrices(name, xs, dtype, shape, device):
    """(list of addresses, leading dimension) of equally shaped matrices."""
    got = [_matrix(f"{name}[{i}]", y, dtype, shape, device) for i, y in enumerate(xs)]
    if len({ld for _, ld in got}) > 1:
        raise ValueError(f"{name}: the matrices' rows lie at different distances")
    return [p for p, _ in got], got[0][1] if got else 1


def muon(w, momentum_buffer, grad, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale=1.0, eps=1e-7, steps=5, copy=None):
    """Updates the matrices `w` and their momenta in place (see b2_muon in include/b200mlp.h): sequences of matrices of one
    shape, or three-dimensional tensors of them. w and momentum_buffer are float32, grad float32 or bfloat16; `copy`, bfloat16,
    receives the new weights too."""
    ws = _listed(w)
    if not ws:
        raise ValueError("w: no matrices")
    shape, device = ws[0].shape, ws[0].device
    ms, gs, cs = _listed(momentum_buffer), _listed(grad), None if copy is None else _listed(copy)
    pw, ldw = _matrices("w", ws, torch.float32, shape, device)
    pm, ldm = _matrices("momentum_buffer", ms, torch.float32, shape, device)
    pg, ldg = _matrices("grad", gs, gs[0].dtype if gs else None, shape, device)
    pc, ldc = _matrices("copy", cs, torch.bfloat16, shape, device) if cs is not None else (None, 0)
    if not len(pw) == len(pm) == len(pg) == (len(pc) if pc is not None else len(pw)):
        raise ValueError("w, momentum_buffer, grad and copy list different numbers of matrices")
    n = len(pw)
    arr = lambda ps: None if ps is None else (C.c_void_p * n)(*ps)  # noqa: E731
    o = K.MuonOptions(lr, momentum, weight_decay, scale, eps, int(nesterov), steps)
    with _on(device) as stream:
        ws_ = _workspace(device, "muon", n, shape[0], shape[1])
        _ck(K.lib().b2_muon(n, shape[0], shape[1], _DTYPES[gs[0].dtype], arr(pw), ldw, arr(pc), ldc, arr(pm), ldm, arr(pg), ldg,
                            C.byref(o), ws_.data_ptr(), ws_.numel(), stream))
    _changed(ws + ms + (cs or []))


def sync(device=None):
    """Waits for the current stream of `device`; K.B2Error with code ERR_TIMEOUT if a bounded wait of a kernel on the device gave up
    since this stream last asked (see b2_lm_sync in include/b200mlp.h)."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"device: {device}, wanted a CUDA device")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with _on(device) as stream:
        _ck(K.lib().b2_lm_sync(stream))
