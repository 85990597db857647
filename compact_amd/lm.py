"""The operators of a language model's training step around its FFN: embedding
lookup with its gradient, the residual norm between blocks, and distillation
from a teacher's top logits.

  embedding, embedding_backward            EmbeddingFunction, ScaledEmbedding
  residual_norm, residual_norm_backward    ResidualNormFunction, ResidualNorm
  distill_topk                             DistillTopKFunction, distill_loss

The lower-case wrappers launch the kernels and take part in no autograd graph,
as those of kernels.py; the Functions and modules do.  float32, float16 and
bfloat16 tensors of any row length and alignment; sums and statistics are
fp32, each output is rounded once.  The reference leaves these operators to
torch.  There is no CPU path.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from ._lib import check
from .kernels import _DT, _dtype_code, _ptr, _require_device, _stream, _timed

_INDEX = {torch.int32: 0, torch.int64: 1}
_GATE_NONE, _GATE_CHANNEL, _GATE_SEQUENCE, _GATE_TOKEN = range(4)
_REDUCTION = {"mean": 0, "sum": 1, "none": 2}


def _index_code(t: torch.Tensor, what: str) -> int:
    assert t.dtype in _INDEX, f"{what}: int32 or int64 expected, got {t.dtype}"
    return _INDEX[t.dtype]


def _on_device(first, *rest):
    """All tensors (None: absent) on one HIP device."""
    dev = first.get_device()
    if dev < 0:
        _require_device(first)
    for t in rest:
        if t is not None and t.get_device() != dev:
            _require_device(t)
            raise AssertionError(f"tensors on {first.device} and {t.device}")


def _new_like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t, d):
    """(tensor, elements between rows) of t seen as [rows, d] with whole rows."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, d
    t = t.reshape(-1, d)
    if t.stride(1) != 1 and d > 1:
        t = t.contiguous()
    return t, t.stride(0)


class _Once(torch.autograd.Function):
    """The first `n` of the tensors themselves: new gradients, as a function of them all
    that cannot be differentiated.  No views, which may not be changed in place."""

    @staticmethod
    def forward(ctx, what, n, *tensors):
        ctx.what = what
        ctx.mark_dirty(*[t for t in tensors[:n] if t is not None])
        return tensors[:n]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.what} is differentiable once: its gradient has no gradient")


def _differentiable_once(what, grads, *inputs):
    """What a Function's backward returns: the gradients that a kernel computed from
    `inputs`.  Under create_graph they are tied to the inputs, so that a second
    derivative through them is an error and no term of it is left out."""
    if not torch.is_grad_enabled():
        return grads
    return _Once.apply(what, len(grads), *grads, *inputs)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------

def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * weight[ids]: [*ids.shape, D] in weight's dtype.  ids: int32 or
    int64; an id outside the table gives a row of zeros."""
    _on_device(weight, ids)
    assert weight.dim() == 2, f"weight [V, D] expected, got {tuple(weight.shape)}"
    wide = _index_code(ids, "ids")
    dt = _dtype_code(weight)
    weight, ids = weight.contiguous(), ids.contiguous()
    v, d = weight.shape
    out = weight.new_empty((*ids.shape, d))
    with _timed("embedding"):
        rc = _lib.api().cpt_embedding(dt, weight.data_ptr(), v, d, ids.data_ptr(), wide,
                                      ids.numel(), float(scale), out.data_ptr(), _stream(weight))
    check(rc, "embedding")
    return out


def embedding_backward(grad: torch.Tensor, ids: torch.Tensor, num_embeddings: int,
                       scale: float = 1.0, *, padding_idx: int | None = None, out=None):
    """The table's gradient of `embedding`: [num_embeddings, D] in grad's dtype,
    row v the fp32 sum of scale * grad over the tokens with id v, added in the
    tokens' order (the same bits on every run).  padding_idx and ids outside the
    table add nothing.  `out` [num_embeddings, D], in grad's dtype or float32,
    is added to instead (a gradient accumulated over micro-batches): only the
    rows that the tokens name are read and written."""
    _on_device(grad, ids, out)
    wide = _index_code(ids, "ids")
    dt = _dtype_code(grad)
    assert grad.dim() >= 1 and grad.shape[:-1] == ids.shape, \
        f"grad {tuple(grad.shape)} for ids {tuple(ids.shape)}"
    d, n, v = grad.shape[-1], ids.numel(), int(num_embeddings)
    assert v >= 0, f"num_embeddings={v}"
    pad = -1
    if padding_idx is not None:
        assert -v <= padding_idx < v, f"padding_idx={padding_idx} outside a table of {v}"
        pad = padding_idx % v
    grad, ld = _rows(grad, d)
    ids = ids.contiguous()
    accumulate = out is not None
    if accumulate:
        assert tuple(out.shape) == (v, d) and out.is_contiguous(), \
            f"out: contiguous {(v, d)} expected, got {tuple(out.shape)}"
        assert out.dtype in (grad.dtype, torch.float32), \
            f"out: {grad.dtype} or float32 expected, got {out.dtype}"
    else:
        out = torch.empty((v, d), dtype=grad.dtype, device=grad.device)
    L = _lib.api()
    nbytes = L.cpt_embedding_backward_workspace_bytes(n, v, d)
    assert nbytes >= 0, f"embedding_backward: {n} tokens, table {(v, d)} out of range"
    ws = torch.empty(nbytes, dtype=torch.uint8, device=grad.device) if nbytes else None
    with _timed("embedding_backward"):
        rc = L.cpt_embedding_backward(dt, _DT[out.dtype], grad.data_ptr(), ld, ids.data_ptr(),
                                      wide, n, v, d, pad, float(scale), int(accumulate),
                                      out.data_ptr(), _ptr(ws), _stream(grad))
    check(rc, "embedding_backward")
    return out


class EmbeddingFunction(torch.autograd.Function):
    """scale * weight[ids] with the table's gradient by sorted tokens; differentiable
    once."""

    @staticmethod
    def forward(ctx, ids, weight, scale=1.0, padding_idx=None):
        ctx.save_for_backward(ids)
        ctx.meta = (weight.shape[0], scale, padding_idx)
        return embedding(ids, weight, scale)

    @staticmethod
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        v, scale, padding_idx = ctx.meta
        dw = None
        if ctx.needs_input_grad[1]:
            dw = embedding_backward(grad, ids, v, scale, padding_idx=padding_idx)
            dw, = _differentiable_once("EmbeddingFunction", (dw,), grad)
        return None, dw, None, None


class ScaledEmbedding(nn.Embedding):
    """nn.Embedding whose output is scaled by `scale`."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale: float = 1.0,
                 device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx=None,
                        scale: float = 1.0):
        """A module over the table `embeddings` [V, D] itself, trained unless `freeze`."""
        assert embeddings.dim() == 2, f"table [V, D] expected, got {tuple(embeddings.shape)}"
        m = cls(*embeddings.shape, padding_idx, scale, device="meta")
        m.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return m

    def extra_repr(self):
        return f"{super().extra_repr()}, scale={self.scale}"

    def forward(self, ids):
        return EmbeddingFunction.apply(ids, self.weight, self.scale, self.padding_idx)


# ---------------------------------------------------------------------------
# residual norm
# ---------------------------------------------------------------------------

def _gate_kind(gate, shape):
    """How a gate broadcasts to [*lead, D]: (kind, rows that share a gate row)."""
    rows = 1
    for s in shape[:-1]:
        rows *= s
    if gate is None:
        return _GATE_NONE, rows
    d = shape[-1]
    lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape[:-1])
    if gate.dim() >= 1 and len(lead) == len(shape) - 1:
        if gate.shape[-1] == d and all(s == 1 for s in lead):
            return _GATE_CHANNEL, rows
        if gate.shape[-1] == 1 and lead == tuple(shape[:-1]):
            return _GATE_TOKEN, rows
        if gate.shape[-1] == d and len(lead) >= 2 and lead[0] == shape[0] \
                and all(s == 1 for s in lead[1:]):
            return _GATE_SEQUENCE, (rows // shape[0] if shape[0] else 0)
    raise AssertionError(f"gate {tuple(gate.shape)} for activations {tuple(shape)}: "
                         "[D], [B, 1, D] or [..., 1] expected")


def _norm_args(x, y, w_pre, w_post, gate, residual_scale):
    """Checks shared by both directions; returns the weights' type code."""
    shape = x.shape
    if y is None:
        assert w_post is None and gate is None and residual_scale == 1.0, \
            "w_post, gate and residual_scale belong to a block's output y"
    else:
        assert y.shape == shape and y.dtype == x.dtype, "residual and y share shape and dtype"
    wdt = x.dtype
    first = w_pre if w_pre is not None else w_post if w_post is not None else gate
    if first is not None:
        wdt = first.dtype
        assert wdt == x.dtype or wdt == torch.float32, \
            f"weights of {wdt} with activations of {x.dtype}"
    for w in (w_pre, w_post):
        assert w is None or (w.dtype == wdt and w.dim() == 1 and w.shape[0] == shape[-1]), \
            f"weights: {wdt} {(shape[-1],)} expected, got {w.dtype} {tuple(w.shape)}"
    assert gate is None or gate.dtype == wdt, "w_pre, w_post and gate share one dtype"
    return _DT[wdt]


def _dense(t):
    return None if t is None else t.contiguous()


def residual_norm(residual, y=None, w_pre=None, *, w_post=None, gate=None, scale: float = 1.0,
                  residual_scale: float = 1.0, eps: float = 1e-6):
    """What lies between two blocks, over the last axis of [..., D]:

        u = y / rms(y) * w_post                       (w_post None: u = y)
        residual_out = residual_scale * residual + scale * gate * u
        x = residual_out / rms(residual_out) * w_pre  (w_pre None: x is None)

    with rms(t) = sqrt(mean t^2 + eps).  gate: None, [D], [B, 1, D] or one value
    per token [..., 1].  Weights and gate share one dtype, the activations' or
    float32.  y None: x is the norm of `residual`, returned as it is.  Returns
    (residual_out, x, stats); stats, fp32 [2, rows], is what the backward
    needs."""
    _on_device(residual, y, w_pre, w_post, gate)
    dt = _dtype_code(residual)
    assert residual.dim() >= 1 and residual.shape[-1] > 0, "residual_norm: [..., D] expected"
    assert y is not None or w_pre is not None, "residual_norm: y or w_pre expected"
    assert eps >= 0, f"eps={eps}"
    wdt = _norm_args(residual, y, w_pre, w_post, gate, residual_scale)
    shape = residual.shape
    d = shape[-1]
    kind, seq = _gate_kind(gate, shape)
    rows = residual.numel() // d
    w_pre, w_post, gate = _dense(w_pre), _dense(w_post), _dense(gate)
    res, ld_res = _rows(residual, d)
    y2, ld_y = _rows(y, d)
    out = _new_like(residual) if y is not None else None
    x = _new_like(residual) if w_pre is not None else None
    stats = torch.empty((2, rows), dtype=torch.float32, device=residual.device)
    if rows == 0:
        return (residual if out is None else out), x, stats
    with _timed("residual_norm"):
        rc = _lib.api().cpt_residual_norm(
            dt, wdt, res.data_ptr(), ld_res, _ptr(y2), ld_y, _ptr(w_post), _ptr(w_pre),
            _ptr(gate), kind, rows, seq, d, float(scale), float(residual_scale), float(eps),
            _ptr(out), _ptr(x), stats.data_ptr(), _stream(residual))
    check(rc, "residual_norm")
    return (residual if out is None else out), x, stats


def residual_norm_backward(d_residual_out, d_x, residual_out, y, stats, w_pre=None, *,
                           w_post=None, gate=None, scale: float = 1.0,
                           residual_scale: float = 1.0):
    """The gradients of `residual_norm` from those of its residual_out (None:
    zeros) and x (None without w_pre), given residual_out, y and stats of the
    forward.  Returns (d_residual, d_y, d_w_pre, d_w_post, d_gate), None for
    what the forward had none of."""
    _on_device(residual_out, d_residual_out, d_x, y, stats, w_pre, w_post, gate)
    dt = _dtype_code(residual_out)
    shape, d = residual_out.shape, residual_out.shape[-1]
    assert (d_x is None) == (w_pre is None), "d_x and w_pre belong together"
    assert y is not None or d_x is not None, "residual_norm_backward: y or d_x expected"
    for t in (d_residual_out, d_x):
        assert t is None or (t.shape == shape and t.dtype == residual_out.dtype), \
            "gradients share residual_out's shape and dtype"
    wdt = _norm_args(residual_out, y, w_pre, w_post, gate, residual_scale)
    kind, seq = _gate_kind(gate, shape)
    rows = residual_out.numel() // d
    assert tuple(stats.shape) == (2, rows) and stats.dtype == torch.float32 \
        and stats.is_contiguous(), f"stats: contiguous float32 {(2, rows)} expected"
    w_pre, w_post, gate = _dense(w_pre), _dense(w_post), _dense(gate)
    d_res = _new_like(residual_out)
    d_y = _new_like(residual_out) if y is not None else None
    make = torch.empty_like if rows else torch.zeros_like
    d_w_pre = None if w_pre is None else make(w_pre)
    d_w_post = None if w_post is None else make(w_post)
    d_gate = None if gate is None else make(gate)
    if rows == 0:
        return d_res, d_y, d_w_pre, d_w_post, d_gate
    dro, ld_dro = _rows(d_residual_out, d)
    dx, ld_dx = _rows(d_x, d)
    ro, ld_ro = _rows(residual_out, d)
    y2, ld_y = _rows(y, d)
    L = _lib.api()
    nbytes = L.cpt_residual_norm_backward_workspace_bytes(rows, seq, d, kind)
    assert nbytes >= 0, f"residual_norm_backward: D={d} out of range"
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=residual_out.device)
    with _timed("residual_norm_backward"):
        rc = L.cpt_residual_norm_backward(
            dt, wdt, _ptr(dro), ld_dro, _ptr(dx), ld_dx, ro.data_ptr(), ld_ro, _ptr(y2),
            ld_y, stats.data_ptr(), _ptr(w_post), _ptr(w_pre), _ptr(gate), kind, rows, seq, d,
            float(scale), float(residual_scale), d_res.data_ptr(), _ptr(d_y), _ptr(d_w_pre),
            _ptr(d_w_post), _ptr(d_gate), ws.data_ptr(), _stream(residual_out))
    check(rc, "residual_norm_backward")
    return d_res, d_y, d_w_pre, d_w_post, d_gate


class ResidualNormFunction(torch.autograd.Function):
    """residual_norm as an autograd Function: (residual_out, x) of (residual, y,
    ...), or with y None (residual, x); x is None without w_pre.  Saves
    residual_out, y and two fp32 values a token.  Differentiable once."""

    @staticmethod
    def forward(ctx, residual, y, w_pre, w_post=None, gate=None, scale=1.0, residual_scale=1.0,
                eps=1e-6):
        out, x, stats = residual_norm(residual, y, w_pre, w_post=w_post, gate=gate, scale=scale,
                                      residual_scale=residual_scale, eps=eps)
        ctx.save_for_backward(out, y, stats, w_pre, w_post, gate)
        ctx.meta = (scale, residual_scale)
        ctx.set_materialize_grads(False)
        return out if y is not None else out.view_as(out), x

    @staticmethod
    def backward(ctx, d_out, d_x):
        out, y, stats, w_pre, w_post, gate = ctx.saved_tensors
        scale, residual_scale = ctx.meta
        if d_out is None and d_x is None:
            return (None,) * 8
        if w_pre is not None and d_x is None:   # x unused: nothing through its norm
            if y is None:
                return d_out, None, torch.zeros_like(w_pre), None, None, None, None, None
            d_x = torch.zeros_like(out)
        grads = residual_norm_backward(d_out, d_x, out, y, stats, w_pre, w_post=w_post, gate=gate,
                                       scale=scale, residual_scale=residual_scale)
        return *_differentiable_once("ResidualNormFunction", grads, d_out, d_x, out, y, w_pre,
                                     w_post, gate), None, None, None


class ResidualNorm(nn.Module):
    """The residual norm between two blocks: (residual, y) -> (residual_out, x),
    x the next block's input.  `post` norms the block's output first (sandwich
    norms), `gate` "channel" learns one factor per channel, starting at
    `gate_init`; another gate ([B, 1, D], [..., 1]) is passed to forward."""

    def __init__(self, dim: int, post: bool = False, pre: bool = True, gate: str | None = None,
                 gate_init: float = 1.0, scale: float = 1.0, residual_scale: float = 1.0,
                 eps: float = 1e-6, device=None, dtype=None):
        super().__init__()
        assert gate in (None, "channel"), f"gate={gate!r}: None or 'channel' expected"
        kw = dict(device=device, dtype=dtype)
        self.w_pre = nn.Parameter(torch.ones(dim, **kw)) if pre else None
        self.w_post = nn.Parameter(torch.ones(dim, **kw)) if post else None
        self.gate = nn.Parameter(torch.full((dim,), float(gate_init), **kw)) if gate else None
        self.scale, self.residual_scale, self.eps = scale, residual_scale, eps

    def forward(self, residual, y=None, gate=None):
        assert gate is None or self.gate is None, "two gates"
        assert gate is None or y is not None, "a gate belongs to a block's output y"
        if y is None:
            return ResidualNormFunction.apply(residual, None, self.w_pre, None, None, 1.0, 1.0,
                                              self.eps)
        return ResidualNormFunction.apply(residual, y, self.w_pre, self.w_post,
                                          self.gate if gate is None else gate, self.scale,
                                          self.residual_scale, self.eps)


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------

def distill_topk(logits, top_logits, top_indices, labels=None, *, top_lse=None,
                 temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                 reduction: str = "mean", grad_out=None, want_grad: bool = True,
                 inplace: bool = False):
    """Distillation from a teacher's top-K logits and its gradient, in one pass
    over the student's logits [..., V]:

        q = softmax(logits / T);  p = softmax(top_logits / T) over the K entries
        soft = T^2 * sum p (log p - log q[top_indices]);  hard = cross entropy
        loss = alpha * soft + (1 - alpha) * hard

    top_lse [...]: the teacher's log-sum-exp of all its logits / T; then
    p = exp(top_logits / T - top_lse), and what it leaves (1 - sum p) is held
    against what q leaves outside the entries (nothing only where all of that is
    -inf: finite logits count, however low).  top_indices: int32 or int64; an
    index outside [0, V) is no entry, and a row without entries has no soft term.
    Rows labelled ignore_index, or outside [0, V), have no loss and a zero
    gradient; alpha < 1 needs labels.  "mean" is over the rows left in (0 where
    there are none).

    Returns (loss fp32, grad in logits' dtype or None): the gradient of the
    reduced loss times grad_out (a number, or a float32 tensor: a scalar, or for
    "none" one value per row).  `inplace` writes it over logits, which must be
    the caller's own.  A row-strided view such as logits[:, :-1] is read as it
    lies."""
    _on_device(logits, top_logits, top_indices, labels, top_lse)
    dt, tdt = _dtype_code(logits), _dtype_code(top_logits)
    assert logits.dim() >= 1 and logits.shape[-1] > 0, "distill_topk: logits [..., V] expected"
    assert reduction in _REDUCTION, f"reduction={reduction!r}"
    assert temperature > 0, f"temperature={temperature}"
    assert alpha == 1.0 or labels is not None, "alpha < 1 needs labels"
    lead, v = logits.shape[:-1], logits.shape[-1]
    assert top_logits.shape == top_indices.shape and top_logits.dim() >= 1 \
        and top_logits.shape[:-1] == lead, \
        f"top_logits {tuple(top_logits.shape)}, top_indices {tuple(top_indices.shape)} for " \
        f"logits {tuple(logits.shape)}"
    k = top_logits.shape[-1]
    wide = _index_code(top_indices, "top_indices")
    label_wide = 0
    if labels is not None:
        assert labels.shape == lead, f"labels {tuple(labels.shape)} for {tuple(logits.shape)}"
        label_wide = _index_code(labels, "labels")
        labels = labels.contiguous()
    if top_lse is not None:
        assert top_lse.shape == lead, f"top_lse {tuple(top_lse.shape)} for {tuple(logits.shape)}"
        top_lse = top_lse.float().contiguous()
    top_logits, top_indices = top_logits.contiguous(), top_indices.contiguous()
    rows = logits.numel() // v

    # rows per batch entry, and the strides of both
    z, seq, ld_b, ld_s = logits, max(rows, 1), 0, v
    if not z.is_contiguous():
        if z.dim() == 2 and (v == 1 or z.stride(1) == 1):
            ld_s = z.stride(0)
        elif z.dim() == 3 and (v == 1 or z.stride(2) == 1):
            seq, ld_b, ld_s = max(z.shape[1], 1), z.stride(0), z.stride(1)
        else:
            z = z.contiguous()
    grad, gld_b, gld_s = None, 0, 0
    if want_grad and inplace:
        assert z is logits and (seq <= 1 or ld_s >= v) and \
            (rows <= seq or ld_b >= (seq - 1) * ld_s + v), \
            "inplace: logits of separate rows, whole along the vocabulary, expected"
        grad, gld_b, gld_s = logits, ld_b, ld_s
    elif want_grad:
        grad = _new_like(logits)
        gld_b, gld_s = seq * v, v
    scale, gout = 1.0, None
    if isinstance(grad_out, torch.Tensor):
        _on_device(logits, grad_out)
        assert grad_out.dtype == torch.float32 and grad_out.numel() == \
            (rows if reduction == "none" else 1), \
            f"grad_out: float32 of the loss's shape expected, got {tuple(grad_out.shape)}"
        gout = grad_out.contiguous()
    elif grad_out is not None:
        scale = float(grad_out)
    # a row's loss each, then (one more) their sum or mean
    losses = torch.empty(rows + 1, dtype=torch.float32, device=logits.device)
    loss = losses[:rows].view(lead) if reduction == "none" else losses[rows]
    with _timed("distill_topk"):
        rc = _lib.api().cpt_distill_topk(
            dt, z.data_ptr(), rows, v, seq, ld_b, ld_s, tdt, top_logits.data_ptr(), wide,
            top_indices.data_ptr(), k, _ptr(top_lse), label_wide, _ptr(labels), ignore_index,
            float(temperature), float(alpha), _REDUCTION[reduction], scale, _ptr(gout),
            losses.data_ptr(), losses.data_ptr() + 4 * rows, _ptr(grad), gld_b, gld_s,
            _stream(logits))
    check(rc, "distill_topk")
    if grad is logits:      # autograd refuses a graph that still needs the old values
        torch.autograd.graph.increment_version(logits)
    return loss, grad


def _scale_rows(x, factor, per_row):
    """x [..., V] *= factor (fp32, one or one per row), skipping factors of 1."""
    v = x.shape[-1]
    check(_lib.api().cpt_scale_rows(_dtype_code(x), x.data_ptr(), x.numel() // v, v,
                                    factor.data_ptr(), int(per_row), _stream(x)), "scale_rows")
    return x


class DistillTopKFunction(torch.autograd.Function):
    """distill_topk's loss with its gradient for the logits.

    bfloat16 and float32: the forward computes the gradient in the pass that
    reads the logits (one read, one write), and the backward multiplies it by
    the loss's incoming gradient, which touches nothing where that is 1; another
    factor than a power of two rounds a second time.  float16: a mean's gradient
    underflows before a loss scale reaches it, so the backward computes it from
    the logits with the incoming gradient.  One backward per forward; differentiable
    once, so create_graph is refused."""

    @staticmethod
    def forward(ctx, logits, top_logits, top_indices, labels=None, top_lse=None, temperature=1.0,
                alpha=1.0, ignore_index=-100, reduction="mean", inplace=False):
        ctx.kw = dict(temperature=temperature, alpha=alpha, ignore_index=ignore_index,
                      reduction=reduction)
        ctx.inplace, ctx.done = inplace, False
        now = ctx.needs_input_grad[0] and logits.dtype != torch.float16
        loss, grad = distill_topk(logits, top_logits, top_indices, labels, top_lse=top_lse,
                                  want_grad=now, inplace=inplace and now, **ctx.kw)
        if now:
            ctx.grad = grad
        elif ctx.needs_input_grad[0]:
            ctx.grad = None
            ctx.save_for_backward(logits, top_logits, top_indices, labels, top_lse)
        return loss

    @staticmethod
    def backward(ctx, grad_out):
        if ctx.done:
            raise RuntimeError("DistillTopKFunction: one backward per forward")
        if torch.is_grad_enabled():     # the logits may be gone: nothing to tie it to
            raise RuntimeError("DistillTopKFunction is differentiable once: no create_graph")
        ctx.done = True
        grad_out = grad_out.float().contiguous()
        if ctx.grad is None:
            logits, top_logits, top_indices, labels, top_lse = ctx.saved_tensors
            _, grad = distill_topk(logits, top_logits, top_indices, labels, top_lse=top_lse,
                                   grad_out=grad_out, inplace=ctx.inplace, **ctx.kw)
        else:
            grad, ctx.grad = ctx.grad, None
            if grad.is_contiguous():
                _scale_rows(grad, grad_out, ctx.kw["reduction"] == "none")
            else:
                grad.mul_(grad_out.unsqueeze(-1) if grad_out.dim() else grad_out)
        return (grad,) + (None,) * 9


def distill_loss(logits, top_logits, top_indices, labels=None, *, top_lse=None,
                 temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                 reduction: str = "mean", inplace: bool = False):
    """distill_topk's loss, differentiable in the logits.  `inplace` lets the
    gradient take the logits' memory (logits must not be read afterwards)."""
    return DistillTopKFunction.apply(logits, top_logits, top_indices, labels, top_lse, temperature,
                                     alpha, ignore_index, reduction, inplace)
