"""Scoring: the log probabilities of given tokens, each row's entropy and its
likeliest alternatives, in one read of the logits.

  token_logprobs, token_logprobs_backward    TokenLogprobsFunction, token_scores

The lower-case wrappers launch the kernels and take part in no autograd graph;
TokenLogprobsFunction and token_scores do.  float32, float16 and bfloat16 logits
of any vocabulary and alignment; statistics are fp32.  The reference leaves this
to torch.  There is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check
from .kernels import _dtype_code, _guard, _ptr, _stream, _timed
from .lm import _differentiable_once, _index_code, _new_like, _on_device

MAX_TOP = 128


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns; fp32 of the logits' leading shape, top_* one axis
    more.  stats [2, rows], where asked for: each row's maximum and the log of its sum,
    which the backward takes in the place of lse where that is too coarse (logits in the
    thousands)."""
    logprobs: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]
    stats: Optional[torch.Tensor]


def _logit_rows(z):
    """logits [..., V] as the kernels read them: (z, rows, rows a batch entry, elements
    between entries and rows)."""
    v = z.shape[-1]
    rows = z.numel() // v
    if not z.is_contiguous():
        if z.dim() == 2 and (v == 1 or z.stride(1) == 1):
            return z, rows, max(rows, 1), 0, z.stride(0)
        if z.dim() == 3 and (v == 1 or z.stride(2) == 1):
            return z, rows, max(z.shape[1], 1), z.stride(0), z.stride(1)
        z = z.contiguous()
    return z, rows, max(rows, 1), 0, v


def _targets(logits, targets):
    if targets is None:
        return None, 0
    assert targets.shape == logits.shape[:-1], \
        f"targets {tuple(targets.shape)} for logits {tuple(logits.shape)}"
    return targets.contiguous(), _index_code(targets, "targets")


def _check_logits(logits, temperature):
    assert logits.dim() >= 1 and logits.shape[-1] > 0, "logits [..., V] expected"
    assert 0 < temperature < float("inf"), f"temperature={temperature}"
    return _dtype_code(logits)


def token_logprobs(logits, targets=None, *, temperature: float = 1.0, top_k: int = 0,
                   ignore_index: int = -100, stats: bool = False) -> TokenLogprobs:
    """Over rows of logits [..., V] with p = softmax(logits / temperature): log
    p[targets], the entropy -sum p log p, the log-sum-exp of logits / temperature, and
    the top_k <= 128 largest log p with their columns (int64), in falling order, equal
    logits by rising column; with `stats` what a backward needs besides.

    targets: int32 or int64 [...], or None (no logprobs).  Rows whose target is
    ignore_index or outside [0, V) are left out: zeros, and alternatives of -inf at
    column -1.  A row of -inf alone has entropy 0 and log probabilities of -inf; a row
    with NaN or +inf is NaN, and its alternatives take NaN for the largest.  A
    row-strided view such as logits[:, :-1] is read as it lies."""
    _on_device(logits, targets)
    dt = _check_logits(logits, temperature)
    targets, wide = _targets(logits, targets)
    lead, v = logits.shape[:-1], logits.shape[-1]
    top_k = int(top_k)
    assert 0 <= top_k <= min(v, MAX_TOP), f"top_k={top_k} of {v} (at most {MAX_TOP})"
    z, rows, seq, ld_b, ld_s = _logit_rows(logits)
    new = logits.new_empty
    logp = kept = None
    if stats:       # for an autograd graph, whose tensors are no views of one another
        if targets is not None:
            logp = new(lead, dtype=torch.float32)
        entropy, lse = new(lead, dtype=torch.float32), new(lead, dtype=torch.float32)
        kept = new((2, rows), dtype=torch.float32)
    elif targets is not None:
        logp, entropy, lse = new((3, *lead), dtype=torch.float32).unbind()
    else:
        entropy, lse = new((2, *lead), dtype=torch.float32).unbind()
    top_p = top_i = None
    if top_k:
        top = (*lead, top_k)
        top_p, top_i = new(top, dtype=torch.float32), new(top, dtype=torch.int64)
    with _guard(logits), _timed("token_logprobs"):
        rc = _lib.api().cpt_token_logprobs(
            dt, z.data_ptr(), rows, v, seq, ld_b, ld_s, wide, _ptr(targets), ignore_index,
            float(temperature), top_k, _ptr(logp), entropy.data_ptr(), lse.data_ptr(),
            _ptr(kept), _ptr(top_p), _ptr(top_i), _stream(logits))
    check(rc, "token_logprobs")
    return TokenLogprobs(logp, entropy, lse, top_p, top_i, kept)


def token_logprobs_backward(logits, targets, lse, entropy, d_logprobs=None, d_entropy=None, *,
                            stats=None, temperature: float = 1.0, ignore_index: int = -100,
                            inplace: bool = False):
    """The logits' gradient, in their dtype, from those of token_logprobs' logprobs and
    entropy (fp32 [...], None: zeros), given lse (or stats) and entropy of the forward.
    Rows left out, and rows of -inf alone, have a gradient of zeros.  `inplace` writes it
    over logits, which must be the caller's own."""
    _on_device(logits, targets, lse, entropy, d_logprobs, d_entropy, stats)
    dt = _check_logits(logits, temperature)
    targets, wide = _targets(logits, targets)
    lead, v = logits.shape[:-1], logits.shape[-1]
    assert d_logprobs is None or targets is not None, "d_logprobs needs targets"
    assert d_entropy is None or entropy is not None, "d_entropy needs entropy"
    assert lse is not None or stats is not None, "lse or stats expected"
    rows_of = []
    for t in (lse, entropy, d_logprobs, d_entropy):
        assert t is None or (t.shape == lead and t.dtype == torch.float32), \
            f"fp32 {tuple(lead)} expected, got {t.dtype} {tuple(t.shape)}"
        rows_of.append(None if t is None else t.contiguous())
    lse, entropy, d_logprobs, d_entropy = rows_of
    z, rows, seq, ld_b, ld_s = _logit_rows(logits)
    if stats is not None:
        assert tuple(stats.shape) == (2, rows) and stats.dtype == torch.float32 \
            and stats.is_contiguous(), f"stats: contiguous float32 {(2, rows)} expected"
    if inplace:
        assert z is logits and (seq <= 1 or ld_s >= v) and \
            (rows <= seq or ld_b >= (seq - 1) * ld_s + v), \
            "inplace: logits of separate rows, whole along the vocabulary, expected"
        grad, gld_b, gld_s = logits, ld_b, ld_s
    else:
        grad, gld_b, gld_s = _new_like(logits), seq * v, v
    with _guard(logits), _timed("token_logprobs_backward"):
        rc = _lib.api().cpt_token_logprobs_backward(
            dt, z.data_ptr(), rows, v, seq, ld_b, ld_s, wide, _ptr(targets), ignore_index,
            float(temperature), _ptr(lse), _ptr(stats), _ptr(entropy), _ptr(d_logprobs),
            _ptr(d_entropy), grad.data_ptr(), gld_b, gld_s, _stream(logits))
    check(rc, "token_logprobs_backward")
    if inplace:      # autograd refuses a graph that still needs the old values
        torch.autograd.graph.increment_version(logits)
    return grad


class TokenLogprobsFunction(torch.autograd.Function):
    """token_logprobs, differentiable in the logits through logprobs and entropy:
    (logprobs, entropy, lse, top_logprobs, top_indices).  The gradient is computed in
    the backward, from the logits again; with `inplace` it takes their memory, so
    that there is one backward.  Differentiable once."""

    @staticmethod
    def forward(ctx, logits, targets=None, temperature=1.0, top_k=0, ignore_index=-100,
                inplace=False):
        # a view's root is a leaf, too, if the view is of a parameter
        root = logits if logits._base is None else logits._base
        if inplace and logits.requires_grad and root.is_leaf and root.requires_grad:
            raise RuntimeError("TokenLogprobsFunction: a leaf's gradient cannot take its memory")
        r = token_logprobs(logits, targets, temperature=temperature, top_k=top_k,
                           ignore_index=ignore_index, stats=True)
        ctx.meta = (temperature, ignore_index, inplace)
        ctx.save_for_backward(logits, targets, r.entropy, r.stats)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in r[2:5] if t is not None])
        return tuple(r[:5])

    @staticmethod
    def backward(ctx, d_logprobs, d_entropy, *_):
        logits, targets, entropy, stats = ctx.saved_tensors
        temperature, ignore_index, inplace = ctx.meta
        if d_logprobs is None and d_entropy is None:
            return (None,) * 6
        if inplace and torch.is_grad_enabled():
            raise RuntimeError("TokenLogprobsFunction: no create_graph with inplace")
        grad = token_logprobs_backward(logits, targets, None, entropy, d_logprobs, d_entropy,
                                       stats=stats, temperature=temperature,
                                       ignore_index=ignore_index, inplace=inplace)
        grad, = _differentiable_once("TokenLogprobsFunction", (grad,), logits, d_logprobs,
                                     d_entropy)
        return (grad,) + (None,) * 5


def token_scores(logits, targets=None, *, temperature: float = 1.0, top_k: int = 0,
                 ignore_index: int = -100, inplace: bool = False):
    """token_logprobs' (logprobs, entropy, lse, top_logprobs, top_indices), the first two
    differentiable in the logits.  `inplace` lets the gradient take the logits' memory
    (they must not be read after the backward)."""
    # without gradients nothing is taken: a leaf is then as good as any
    return TokenLogprobsFunction.apply(logits, targets, temperature, top_k, ignore_index,
                                       inplace and torch.is_grad_enabled())
