"""Attention's input: the norms of queries' and keys' heads and their position
rotation in one pass.

  qk_rope, qk_rope_backward    QKRopeFunction, QKNormRope

The lower-case wrappers launch the kernels and take part in no autograd graph;
the Function and the module do.  float32, float16 and bfloat16 heads of any even
width up to 1024, read as they lie (views of one projection's output, heads
before tokens); norms and rotation are fp32 and each output is rounded once.  The
reference leaves these operators to torch.  There is no CPU path.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from ._lib import check
from .kernels import _DT, _dtype_code, _guard, _ptr, _stream, _timed
from .lm import _dense, _differentiable_once, _index_code, _new_like, _on_device


def _strides(t):
    """t [..., S, H, D] with contiguous columns, and the elements between its sequences,
    tokens and heads."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        t = t.contiguous()
        st = t.stride()
    return t, (st[:3] if len(st) == 4 else (0, st[0], st[1]))


def _rope_args(q, k, positions, inv_freq, w_q, w_k, eps):
    """Checks shared by both directions: (batch, seq, q's heads, k's, D, frequencies,
    positions, their code and stride, weights' type)."""
    qs, ks = q.shape, k.shape
    assert len(qs) in (3, 4), f"q [B, S, H, D] or [S, H, D] expected, got {tuple(qs)}"
    *lead, hq, d = qs
    *lead_k, hk, dk = ks
    assert lead == lead_k and d == dk and q.dtype == k.dtype, \
        f"q {q.dtype} {tuple(qs)} and k {k.dtype} {tuple(ks)} share all but their heads"
    assert hq > 0 and hk > 0, "q and k have a head at least"
    assert d % 2 == 0 and d > 0, f"head width {d}: even expected"
    assert inv_freq.dtype == torch.float32 and inv_freq.dim() == 1, \
        f"inv_freq: float32 [R / 2] expected, got {inv_freq.dtype} {tuple(inv_freq.shape)}"
    half = inv_freq.shape[0]
    assert 0 < 2 * half <= d, f"inv_freq: at most {d // 2} frequencies expected, got {half}"
    assert (w_q is None) == (w_k is None), "w_q and w_k belong together"
    assert eps >= 0, f"eps={eps}"
    wdt = q.dtype
    if w_q is not None:
        wdt = w_q.dtype
        assert wdt == q.dtype or wdt == torch.float32, f"weights of {wdt} with heads of {q.dtype}"
        for w in (w_q, w_k):
            assert w.dtype == wdt and w.shape == (d,), \
                f"weights: {wdt} {(d,)} expected, got {w.dtype} {tuple(w.shape)}"
    b, s = lead if len(lead) == 2 else (1, lead[0])
    wide = pos_batch = 0
    if positions is not None:
        wide = _index_code(positions, "positions")
        at = tuple(positions.shape)
        assert at in ((b, s), (1, s), (s,)) and (len(at) == 1 or len(lead) == 2), \
            f"positions {at}: {tuple(lead)} or {(s,)} expected"
        if at == (b, s):
            pos_batch = s
        positions = positions.contiguous()
    return b, s, hq, hk, d, 2 * half, positions, wide, pos_batch, _DT[wdt]


def _nest(strides, shape):
    """Whether an order of the axes nests them: then no two elements share memory."""
    extent = 1
    for stride, size in sorted([(st, n) for st, n in zip(strides, shape) if n > 1]):
        if stride < extent:
            return False
        extent = stride * size
    return True


def _apart(q, k):
    """Whether the elements of q and of k all have places of their own."""
    if q.numel() == 0 or k.numel() == 0:
        return _nest(q.stride(), q.shape) and _nest(k.stride(), k.shape)
    off = (k.data_ptr() - q.data_ptr()) // q.element_size()
    sq, sk = q.stride(), k.stride()
    if q.is_contiguous() and k.is_contiguous():
        return off >= q.numel() or -off >= k.numel()
    same = sq == sk or all([a == b or n == 1 for a, b, n in zip(sq, sk, (*q.shape[:-2], 2, 2))])
    if same and sq[-2] > 0:
        # heads of one buffer: apart if all from the first's to the last's are
        at, rest = divmod(off, sq[-2])
        hq, hk = q.shape[-2], k.shape[-2]
        if rest == 0 and (at >= hq or -at >= hk):
            heads = max(hq, at + hk) - min(0, at)
            if _nest(sq, (*q.shape[:-2], heads, q.shape[-1])):
                return True
    return _nest(sq, q.shape) and _nest(sk, k.shape) and not _meet(off, sq, q.shape, sk, k.shape)


def _meet(off, sq, nq, sk, nk):
    """Whether views with nested axes, `off` elements apart, have elements in one place:
    whether differences of their indices can make up for `off`.  The largest stride first,
    few can; views that would take long to tell apart count as meeting."""
    reach = {}              # how far indices along a stride can differ, both ways
    for st, n in zip(sq, nq):
        if n > 1:
            first, last = reach.get(st, (0, 0))
            reach[st] = first, last + n - 1
    for st, n in zip(sk, nk):
        if n > 1:
            first, last = reach.get(st, (0, 0))
            reach[st] = first - n + 1, last
    axes = sorted([(st, *ends) for st, ends in reach.items()])
    least = sum([st * first for st, first, _ in axes])
    most = sum([st * last for st, _, last in axes])
    if not least <= off <= most:
        return False
    left = {off}
    for st, first, last in reversed(axes):
        # what the smaller strides reach
        least, most = least - st * first, most - st * last
        left = {t - st * n for t in left for n in range(max(first, -((most - t) // st)),
                                                        min(last, (t - least) // st) + 1)}
        if len(left) > 64:
            return True
    return 0 in left


def qk_rope(q: torch.Tensor, k: torch.Tensor, positions, inv_freq: torch.Tensor, *, w_q=None,
            w_k=None, eps: float = 1e-6, interleaved: bool = False, scaling: float = 1.0,
            inplace: bool = False, inverse: bool = False):
    """(q_out, k_out) of q [B, S, H, D] and k [B, S, Hk, D] (or [S, H, D]): heads
    normed where w_q and w_k [D] are given, then turned by their positions:

        n = x / sqrt(mean x^2 + eps) * w
        pairs (a, b) of the first R columns -> scaling * (a cos t - b sin t,
        b cos t + a sin t),  t = position * inv_freq[pair],  R = 2 len(inv_freq)

    A pair is columns i and R / 2 + i, or with `interleaved` 2 i and 2 i + 1; columns
    from R on are normed alone.  positions: int32 or int64 [B, S] or [S], None: 0
    to S - 1; angles are products of 53 bits (1e-7 off at 2 10^9).  Weights share one
    dtype, the heads' or float32.  Outputs are contiguous; `inplace` writes over q and
    k, which must be the caller's own and lie apart.  `inverse` turns back, without
    norms: the gradient."""
    _on_device(q, k, positions, inv_freq, w_q, w_k)
    dt = _dtype_code(q)
    b, s, hq, hk, d, rot, pos, wide, pos_batch, wdt = _rope_args(q, k, positions, inv_freq, w_q,
                                                                 w_k, eps)
    assert not (inverse and w_q is not None), "inverse: of heads without norms"
    inv_freq, w_q, w_k = inv_freq.contiguous(), _dense(w_q), _dense(w_k)
    q2, sq = _strides(q)
    k2, sk = _strides(k)
    if inplace:
        assert q2 is q and k2 is k and _apart(q, k), \
            "inplace: heads with contiguous columns, no two elements in one place, expected"
        q_out, k_out, oq, ok = q, k, sq, sk
    else:
        q_out, k_out = _new_like(q), _new_like(k)
        oq, ok = (s * hq * d, hq * d, d), (s * hk * d, hk * d, d)
    with _guard(q), _timed("qk_rope"):
        rc = _lib.api().cpt_qk_rope(
            dt, wdt, int(interleaved), int(inverse), q2.data_ptr(), *sq, k2.data_ptr(), *sk,
            _ptr(w_q), _ptr(w_k), _ptr(pos), wide, pos_batch, inv_freq.data_ptr(), b, s, hq, hk, d,
            rot, float(eps), float(scaling), q_out.data_ptr(), *oq,
            k_out.data_ptr(), *ok, _stream(q))
    check(rc, "qk_rope")
    if inplace:
        torch.autograd.graph.increment_version((q, k))
    return q_out, k_out


def qk_rope_backward(d_q, d_k, q, k, positions, inv_freq, *, w_q=None, w_k=None,
                     eps: float = 1e-6, interleaved: bool = False, scaling: float = 1.0):
    """The gradients of `qk_rope` from those of its outputs and its inputs:
    (d_q, d_k, d_w_q, d_w_k), the last two None without weights; then q and k
    are not read and may be None."""
    if w_q is None and w_k is None:
        dq, dk = qk_rope(d_q, d_k, positions, inv_freq, interleaved=interleaved, scaling=scaling,
                         inverse=True)
        return dq, dk, None, None
    _on_device(q, k, d_q, d_k, positions, inv_freq, w_q, w_k)
    dt = _dtype_code(q)
    for g, t in ((d_q, q), (d_k, k)):
        assert g.shape == t.shape and g.dtype == t.dtype, "gradients share q's and k's shapes " \
            "and dtype"
    b, s, hq, hk, d, rot, pos, wide, pos_batch, wdt = _rope_args(q, k, positions, inv_freq, w_q,
                                                                 w_k, eps)
    inv_freq, w_q, w_k = inv_freq.contiguous(), _dense(w_q), _dense(w_k)
    q2, sq = _strides(q)
    k2, sk = _strides(k)
    gq, sgq = _strides(d_q)
    gk, sgk = _strides(d_k)
    dq, dk = _new_like(q), _new_like(k)
    if b * s == 0:
        return dq, dk, torch.zeros_like(w_q), torch.zeros_like(w_k)
    dw_q, dw_k = torch.empty_like(w_q), torch.empty_like(w_k)
    L = _lib.api()
    nbytes = L.cpt_qk_rope_backward_workspace_bytes(b * s, hq, hk, d)
    assert nbytes >= 0, f"qk_rope_backward: {tuple(q.shape)} out of range"
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=q.device)
    with _guard(q), _timed("qk_rope_backward"):
        rc = L.cpt_qk_rope_backward(
            dt, wdt, int(interleaved), gq.data_ptr(), *sgq, gk.data_ptr(), *sgk, q2.data_ptr(), *sq,
            k2.data_ptr(), *sk, w_q.data_ptr(), w_k.data_ptr(), _ptr(pos), wide, pos_batch,
            inv_freq.data_ptr(), b, s, hq, hk, d, rot, float(eps),
            float(scaling), dq.data_ptr(), dk.data_ptr(), dw_q.data_ptr(), dw_k.data_ptr(),
            ws.data_ptr(), _stream(q))
    check(rc, "qk_rope_backward")
    return dq, dk, dw_q, dw_k


class QKRopeFunction(torch.autograd.Function):
    """qk_rope as an autograd Function: (q_out, k_out).  With norms it saves q and k
    and computes their statistics again; without, nothing.  Differentiable once."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, w_q=None, w_k=None, eps=1e-6, interleaved=False,
                scaling=1.0):
        ctx.meta = (eps, interleaved, scaling)
        norm = w_q is not None
        ctx.save_for_backward(q if norm else None, k if norm else None, positions, inv_freq, w_q,
                              w_k)
        return qk_rope(q, k, positions, inv_freq, w_q=w_q, w_k=w_k, eps=eps,
                       interleaved=interleaved, scaling=scaling)

    @staticmethod
    def backward(ctx, d_q, d_k):
        q, k, positions, inv_freq, w_q, w_k = ctx.saved_tensors
        eps, interleaved, scaling = ctx.meta
        grads = qk_rope_backward(d_q, d_k, q, k, positions, inv_freq, w_q=w_q, w_k=w_k, eps=eps,
                                 interleaved=interleaved, scaling=scaling)
        dq, dk, dwq, dwk = _differentiable_once("QKRopeFunction", grads, d_q, d_k, q, k, w_q, w_k)
        return dq, dk, None, None, dwq, dwk, None, None, None


class QKNormRope(nn.Module):
    """(q, k) -> (q_out, k_out): heads normed with learned weights (`norm`) and turned
    by their positions.  Frequencies are base^(-2 i / rotary), or those given ([R / 2],
    R = `rotary`); in float32 whatever the module is cast to."""

    def __init__(self, head_dim: int, rotary: int | None = None, base: float = 10000.0,
                 norm: bool = True, eps: float = 1e-6, interleaved: bool = False,
                 scaling: float = 1.0, device=None, dtype=None, inv_freq=None):
        super().__init__()
        if inv_freq is not None:
            assert inv_freq.dim() == 1 and rotary in (None, 2 * inv_freq.numel()), \
                f"inv_freq {tuple(inv_freq.shape)} for rotary={rotary}"
            rotary = 2 * inv_freq.numel()
        self.rotary = head_dim if rotary is None else rotary
        assert 0 < self.rotary <= head_dim and self.rotary % 2 == 0, f"rotary={rotary}"
        self.base, self.eps, self.interleaved, self.scaling = base, eps, interleaved, scaling
        kw = dict(device=device, dtype=dtype)
        self.w_q = nn.Parameter(torch.ones(head_dim, **kw)) if norm else None
        self.w_k = nn.Parameter(torch.ones(head_dim, **kw)) if norm else None
        self._given = None if inv_freq is None else inv_freq.detach().cpu().float()
        self.register_buffer("inv_freq", self._frequencies(device), persistent=False)

    def _frequencies(self, device):
        if self._given is not None:
            return self._given.to(device, copy=True)
        i = torch.arange(0, self.rotary, 2, dtype=torch.float64, device=device)
        return (self.base ** (-i / self.rotary)).float()

    def _apply(self, fn, recurse=True):
        kept = self.inv_freq
        super()._apply(fn, recurse)
        # moved as they are, also where they were changed since: not cast, not left empty
        device = self.inv_freq.device
        self.inv_freq = self._frequencies(device) if kept.is_meta else kept.to(device)
        return self

    def extra_repr(self):
        return f"rotary={self.rotary}, base={self.base}, norm={self.w_q is not None}, " \
               f"interleaved={self.interleaved}"

    def forward(self, q, k, positions=None):
        return QKRopeFunction.apply(q, k, positions, self.inv_freq, self.w_q, self.w_k, self.eps,
                                    self.interleaved, self.scaling)
