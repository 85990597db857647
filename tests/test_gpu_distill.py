"""Distillation from a teacher's top logits against its definition in 64 bits.

Bounds, with e = 2^-24 and u one unit in the output type's last place.  A term
exp((z - max) / tau) has a relative error of (|z - max| / tau + 4) e, sums have
chains of at most 150 terms (the rows read twice: one a vector of a thread), so
with R = 1 + the row's finite range / tau a softmax value and a logarithm's
argument are good to (R + 200) e:
  loss       (R + 400) e * (alpha tau^2 (sum p (|log p| + |log q| + 1) + the same
             of the rest) + (1 - alpha) (|hard| + 1)) + the rest's own error:
             p_rest = 1 - sum p is off by (8 |lse| + 8 + k) e
  gradient   u |exact| + (R + 400) e * the sum of its terms' absolute values
             + the rest's error times q / q_rest
Half-precision gradients are scaled as under a loss scale.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}
E = 2.0 ** -24


def _cpt():
    import compact_amd
    return compact_amd


def definition(z, t, idx, labels, lse, tau, alpha, ignore, reduction, gout):
    """(loss, gradient, loss bound, gradient bound) in 64 bits: a plain dense form."""
    z, t = z.double(), t.double() / tau
    n, v = z.shape
    keep = torch.ones(n, dtype=torch.bool, device=z.device)
    if labels is not None:
        keep = (labels != ignore) & (labels >= 0) & (labels < v)
    entry = (idx >= 0) & (idx < v)
    t = torch.where(entry, t, -math.inf)
    if lse is None:
        base = torch.logsumexp(t, 1, keepdim=True) if t.shape[1] else t.new_zeros(n, 1)
        lp = torch.where(base > -math.inf, t - base, -math.inf)
    else:
        lp = t - lse.double()[:, None]
    p = lp.exp()
    j = idx.clamp(0, v - 1).long()
    lq, l1 = torch.log_softmax(z / tau, 1), torch.log_softmax(z, 1)
    lqj = lq.gather(1, j)
    zero = torch.zeros_like(p)
    soft = torch.where(p > 0, p * (lp - lqj), zero).sum(1)
    size = torch.where(p > 0, p * (lp.abs() + lqj.abs() + 1), zero).sum(1)
    dense = torch.zeros_like(z).scatter_add_(1, j, p)
    top = torch.zeros_like(z).scatter_add_(1, j, entry.double()) > 0
    mass = p.sum(1)
    d = lq.exp() * mass[:, None] - dense
    dsize = lq.exp() * mass[:, None] + dense
    extra, dextra = torch.zeros(n, device=z.device), torch.zeros_like(z)
    if lse is not None:
        off = (8 * lse.double().abs() + 8 + p.shape[1]) * E
        lo = torch.logsumexp(lq.masked_fill(top, -math.inf), 1)
        rest = torch.where(lo > -math.inf, (1 - mass).clamp(min=0), 0.0)
        lrest = torch.where(rest > 0, rest, 1.0).log()
        soft = soft + torch.where(rest > 0, rest * (lrest - lo), 0.0)
        size = size + torch.where(rest > 0, rest * (lrest.abs() + lo.abs() + 1), 0.0)
        # p_rest log p_rest - p_rest log q_rest near p_rest (and below what it is known to)
        some = torch.where(lo > -math.inf, lo.abs(), 0.0)
        extra = off * ((rest + off).log().abs() + 2 + some)
        cond = torch.where(top, 0.0, (lq - lo[:, None]).exp())
        cond = torch.where(lo[:, None] > -math.inf, cond, 0.0)
        d = d + rest[:, None] * (lq.exp() - cond)
        dsize = dsize + rest[:, None] * (lq.exp() + cond)
        dextra = off[:, None] * (lq.exp() + cond)
    loss = alpha * tau ** 2 * soft
    size, extra = alpha * tau ** 2 * size, alpha * tau ** 2 * extra
    d, dsize, dextra = alpha * tau * d, alpha * tau * dsize, alpha * tau * dextra
    if alpha != 1:
        y = torch.where(keep, labels, 0).long()[:, None]
        hard = -l1.gather(1, y)[:, 0]
        hot = torch.zeros_like(z).scatter_(1, y, 1.0)
        loss, size = loss + (1 - alpha) * hard, size + (1 - alpha) * (hard + 1)
        d, dsize = d + (1 - alpha) * (l1.exp() - hot), dsize + (1 - alpha) * (l1.exp() + hot)
    finite = torch.where(z.isfinite() & (z > -1e30), z, z.amax(1, keepdim=True))
    r = 1 + (finite.amax(1) - finite.amin(1)) / min(tau, 1.0)
    bound = (r + 400) * E * size + extra
    dbound = ((r + 400) * E)[:, None] * dsize + dextra
    if lse is not None:      # an entry's p = exp(t - lse) has the exponent's error
        spread = (t - lse.double()[:, None]).abs().masked_fill(~entry | t.isinf(), 0.0).amax(1) \
            if t.shape[1] else torch.zeros_like(r)
        bound = bound + (spread + lse.double().abs()) * E * 4 * size
        dbound = dbound + ((spread + lse.double().abs()) * E * 4)[:, None] * dsize
    zero = torch.zeros_like(loss)
    loss, bound = torch.where(keep, loss, zero), torch.where(keep, bound, zero)
    live = max(1, int(keep.sum()))
    scale = gout if isinstance(gout, torch.Tensor) else torch.full((n,), float(gout))
    scale = scale.double().to(z.device).expand(n) / (live if reduction == "mean" else 1)
    scale = torch.where(keep, scale, zero)[:, None]
    d = torch.where(keep[:, None], d * scale, 0.0)
    dbound = torch.where(keep[:, None], dbound * scale.abs(), 0.0)
    if reduction != "none":
        k = live if reduction == "mean" else 1
        bound = (bound.sum() + 40 * E * loss.abs().sum()) / k
        loss = loss.sum() / k
    return loss, d, bound, dbound


def _close(got, exact, bound, what):
    got = got.double().reshape(exact.shape)
    same = (got == exact) | (got.isnan() & exact.isnan())
    bad = ~((got - exact).abs() <= bound) & ~same
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst " \
        f"{float((got - exact).abs()[bad].max()):.3e}"


def check(z, t, idx, labels=None, lse=None, tau=1.0, alpha=1.0, ignore=-100, reduction="mean",
          gout=1.0, **kw):
    cpt = _cpt()
    v, k = z.shape[-1], t.shape[-1]
    n = z.numel() // v
    want = definition(z.reshape(n, v), t.reshape(n, k), idx.reshape(n, k),
                      None if labels is None else labels.reshape(-1),
                      None if lse is None else lse.reshape(-1), tau, alpha, ignore, reduction,
                      gout.reshape(-1) if isinstance(gout, torch.Tensor) else gout)
    dtype = z.dtype
    loss, grad = cpt.distill_topk(z, t, idx, labels, top_lse=lse, temperature=tau, alpha=alpha,
                                  ignore_index=ignore, reduction=reduction, grad_out=gout, **kw)
    _close(loss, want[0], want[2] + 2.0 ** -23 * want[0].abs(), "loss")
    if grad is not None:
        assert grad.dtype == dtype and grad.shape == z.shape
        _close(grad.reshape(want[1].shape), want[1],
               UNIT[dtype] * want[1].abs() + TINY[dtype] + want[3], "gradient")
    return loss, grad


def _inputs(n, v, k, dtype, device, seed=0, tau=1.0, tail=False, labels=True):
    g = torch.Generator().manual_seed(seed + 7 * n + v + k)
    z = 2 * torch.randn(n, v, generator=g)
    cand = torch.randint(0, v, (n, min(6, v)), generator=g)
    z.scatter_add_(1, cand, 4 + 8 * torch.rand(n, cand.shape[1], generator=g))
    z = z.to(dtype)
    teacher = 0.7 * z.float() + torch.randn(n, v, generator=g)
    top, idx = teacher.topk(k, 1)
    y = cand[:, 0].clone()
    y[torch.rand(n, generator=g) < 0.3] = -100
    lse = torch.logsumexp(teacher.double() / tau, 1).float() if tail else None
    ts = (z, top, idx, y if labels else None, lse)
    return tuple(None if t is None else t.to(device) for t in ts)


# one vector a thread up to rows read twice, odd widths at every step
VOCABS = [1, 7, 64, 1001, 2048, 2051, 4099, 8192, 8209, 16390, 32000, 32769, 50021, 65544, 131099]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", VOCABS)
@pytest.mark.parametrize("mix", ["soft", "soft_tau", "hard", "hard_tau"])
def test_against_definition(device, dtype, v, mix):
    tau = 2.0 if "tau" in mix else 1.0
    alpha = 0.6 if "hard" in mix else 1.0
    gout = 4096.0 if dtype == torch.float16 else 1.0
    for tail in (False, True):
        k = min(v, 13)
        z, t, idx, y, lse = _inputs(9, v, k, dtype, device, tau=tau, tail=tail)
        check(z, t, idx, y, lse, tau, alpha, gout=gout)


@pytest.mark.parametrize("k", [0, 1, 2, 63, 64, 65, 200, 2048])
@pytest.mark.parametrize("tail", [False, True])
def test_entries(device, k, tail):
    z, t, idx, y, lse = _inputs(5, 4099, k, torch.float32, device, tau=1.5, tail=tail)
    check(z, t, idx, y, lse, 1.5, 0.7)
    check(z, t.to(torch.bfloat16), idx.int(), y, lse, 1.5, 0.7)
    check(z, t.half(), idx.int(), y.int(), lse, 1.5, 1.0)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n", [1, 2, 300, 2100])
def test_reductions(device, reduction, n):
    cpt = _cpt()
    z, t, idx, y, lse = _inputs(n, 515, 9, torch.bfloat16, device)
    loss, grad = check(z, t, idx, y, None, 2.0, 0.5, reduction=reduction, gout=0.25)
    assert loss.shape == ((n,) if reduction == "none" else ())
    per_row = torch.rand(n, device=device) if reduction == "none" else torch.tensor(
        3.5, device=device)
    check(z, t, idx, y, None, 2.0, 0.5, reduction=reduction, gout=per_row)
    again = cpt.distill_topk(z, t, idx, y, temperature=2.0, alpha=0.5, reduction=reduction,
                             grad_out=0.25)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    only, none = cpt.distill_topk(z, t, idx, y, temperature=2.0, alpha=0.5, reduction=reduction,
                                  want_grad=False)
    assert none is None and torch.equal(only, loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [520, 40000])
def test_rows_left_out(device, dtype, v):
    """Ignored rows (whatever they hold) and labels outside the vocabulary."""
    z, t, idx, y, lse = _inputs(12, v, 6, dtype, device)
    y[:] = torch.arange(12, device=device)
    y[2], y[5], y[6] = 7, v, -3
    z[2], t[5] = float("nan"), float("nan")
    loss, grad = check(z, t, idx, y, None, 1.0, 0.5, ignore=7)
    for r in (2, 5, 6, 7):
        assert (grad[r] == 0).all()
    y[:] = 7
    loss, grad = check(z, t, idx, y, None, 1.0, 0.5, ignore=7)
    assert loss == 0 and (grad == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("v", [200, 8209, 70001])
def test_masked_columns(device, dtype, tail, v):
    """Logits of -inf and of the type's lowest value; entries masked by either;
    padded, repeated and absent entries; nothing left outside the entries."""
    n, k = 8, 8
    z, t, idx, y, lse = _inputs(n, v, k, dtype, device, tail=tail)
    y[:] = idx[:, 0]
    z[0, v // 2:] = -math.inf
    z[1, v // 2:] = torch.finfo(dtype).min
    z[0, idx[0]], z[1, idx[1]] = 1.0, 2.0
    idx[2, 3:] = -1                          # padding
    idx[3, :] = v + 5                        # no entry at all
    idx[4, 1] = idx[4, 0]                    # an index twice
    t[5, 4:] = -math.inf
    z[6] = -math.inf                         # the student knows the entries only
    z[6, idx[6]] = torch.linspace(0, 3, k, device=device).to(dtype)
    z[7] = torch.finfo(dtype).min            # nothing but the lowest value
    if tail:
        lse[2:5] += 1
    gout = 256.0 if dtype == torch.float16 else 1.0
    loss, grad = check(z, t, idx, y, lse, 1.0, 1.0, gout=gout, reduction="none")
    assert loss.isfinite().all() and grad.isfinite().all()
    check(z, t, idx, y, lse, 1.0, 0.5, gout=gout, reduction="none")


@pytest.mark.parametrize("v", [200, 70001])
def test_not_finite(device, v):
    """An entry on a masked logit costs infinitely much; NaN stays in its row."""
    cpt = _cpt()
    z, t, idx, _, _ = _inputs(4, v, 5, torch.float32, device, labels=False)
    z[0, idx[0, 0]] = -math.inf
    z[1, 3] = math.nan
    z[2, 3] = math.inf
    loss, grad = cpt.distill_topk(z, t, idx, reduction="none")
    assert loss[0] == math.inf and grad[0].isfinite().all()
    assert loss[1].isnan() and grad[1].isnan().any()
    assert loss[2].isnan()
    assert loss[3].isfinite() and grad[3].isfinite().all()


def test_far_below_the_entries(device):
    """What lies outside the entries may be far below them: q_rest keeps its digits."""
    z, t, idx, y, lse = _inputs(3, 3000, 4, torch.float32, device, tail=True)
    z.clamp_(max=5.0)
    z.scatter_add_(1, idx, torch.full((3, 4), 150.0, device=device))
    lse += 0.5
    y[:] = (idx[:, 0] + 1) % 3000
    check(z, t, idx, y, lse, 1.0, 0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(device, dtype):
    """Views read as they lie, and the gradient written over the logits."""
    cpt = _cpt()
    z, t, idx, y, _ = _inputs(20, 1003, 5, dtype, device)
    z3, t3, idx3, y3 = z.view(4, 5, 1003), t.view(4, 5, 5), idx.view(4, 5, 5), y.view(4, 5)
    gout = 512.0 if dtype == torch.float16 else 1.0
    whole = check(z3, t3, idx3, y3, None, 2.0, 0.5, gout=gout)
    shifted = check(z3[:, :-1], t3[:, 1:], idx3[:, 1:], y3[:, 1:], None, 2.0, 0.5, gout=gout)
    check(z3[:, :, 1:900], t3, idx3.clamp(max=800), y3.clamp(max=800), None, 2.0, 0.5, gout=gout)
    check(z3[::2, 1::2], t3[::2, 1::2], idx3[::2, 1::2], y3[::2, 1::2], None, 2.0, 0.5, gout=gout)
    check(z[:, ::2], t, idx.clamp(max=400), None, None, 2.0, 1.0, gout=gout)
    check(z[:1].expand(20, 1003), t, idx, y, None, 2.0, 0.5, gout=gout)
    kw = dict(temperature=2.0, alpha=0.5, grad_out=gout)
    own = z3.clone()
    loss, grad = cpt.distill_topk(own, t3, idx3, y3, inplace=True, **kw)
    assert grad is own and torch.equal(own, whole[1]) and torch.equal(loss, whole[0])
    own = z3.clone()
    loss, grad = cpt.distill_topk(own[:, :-1], t3[:, 1:], idx3[:, 1:], y3[:, 1:], inplace=True,
                                  **kw)
    assert torch.equal(own[:, :-1], shifted[1]) and torch.equal(own[:, -1], z3[:, -1])
    wide = torch.randn(3, 70001, device=device).to(dtype)
    wt, widx = wide.float().topk(4, 1)
    ref = cpt.distill_topk(wide, wt * 2, widx, grad_out=gout)
    loss, grad = cpt.distill_topk(wide, wt * 2, widx, grad_out=gout, inplace=True)
    assert torch.equal(wide, ref[1])


def test_no_rows(device):
    cpt = _cpt()
    z = torch.zeros(0, 50, device=device)
    t, i = torch.zeros(0, 3, device=device), torch.zeros(0, 3, dtype=torch.int64, device=device)
    loss, grad = cpt.distill_topk(z, t, i)
    assert loss == 0 and grad.shape == (0, 50)
    loss, grad = cpt.distill_topk(z, t, i, reduction="none")
    assert loss.shape == (0,)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_function_against_differences(device, dtype, tail):
    """The Function's gradient (scaled by what flows in) along a direction against
    the difference quotient of the 64-bit loss (step 1e-4: truncation ~1e-8)."""
    cpt = _cpt()
    z, t, idx, y, lse = _inputs(6, 300, 7, dtype, device, tau=2.0, tail=tail)
    leaf = z.clone().requires_grad_(True)
    loss = cpt.distill_loss(leaf, t, idx, y, top_lse=lse, temperature=2.0, alpha=0.4)
    (loss * 3000.0).backward()
    step = torch.randn(z.shape, device=device, dtype=torch.float64)
    f = [definition(z.double() + s * 1e-4 * step, t, idx, y, lse, 2.0, 0.4, -100, "mean", 1.0)[0]
         for s in (1, -1)]
    want, got = (f[0] - f[1]) / 2e-4 * 3000.0, (leaf.grad.double() * step).sum()
    size = (leaf.grad.double() * step).abs().sum()
    assert (got - want).abs() <= (1e-5 + UNIT[dtype]) * size


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_function(device, dtype, reduction):
    """Incoming gradients other than 1, memory taken over, a second backward."""
    cpt = _cpt()
    z, t, idx, y, _ = _inputs(8, 2000, 5, dtype, device)
    w = torch.rand(8, device=device) if reduction == "none" else torch.tensor(256.0,
                                                                              device=device)
    want = definition(z, t, idx, y, None, 1.0, 0.5, -100, reduction, w)
    for inplace in (False, True):
        leaf = z.clone().requires_grad_(True)
        logits = leaf * 1
        loss = cpt.distill_loss(logits, t, idx, y, alpha=0.5, reduction=reduction,
                                inplace=inplace)
        total = (loss * w).sum()
        total.backward(retain_graph=True)
        _close(leaf.grad, want[1], 2 * UNIT[dtype] * want[1].abs() + 2 * TINY[dtype] + want[3],
               "gradient")
        with pytest.raises(RuntimeError):
            total.backward()
    with torch.no_grad():
        assert not cpt.distill_loss(z, t, idx, y, alpha=0.5).requires_grad


def test_widest(device):
    """The widest vocabulary with the most entries (96 KiB of LDS)."""
    z, t, idx, y, lse = _inputs(2, 524288, 2048, torch.bfloat16, device, tail=True)
    y[0] = -100
    check(z, t, idx, y, lse, 1.0, 0.5)
    check(z, t, idx, y, None, 2.0, 0.5)


def test_inplace_is_known_to_autograd(device):
    """A graph that keeps the logits themselves cannot be used after they are gone."""
    cpt = _cpt()
    z, t, idx, _, _ = _inputs(4, 300, 5, torch.float32, device, labels=False)
    leaf = z.clone().requires_grad_(True)
    loss = cpt.distill_loss(torch.tanh(leaf), t, idx, inplace=True)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_graph(device):
    """Captured and replayed, with other work between the replays."""
    cpt = _cpt()
    z, t, idx, y, _ = _inputs(40, 5003, 9, torch.bfloat16, device)
    kw = dict(temperature=2.0, alpha=0.5)
    cpt.distill_topk(z, t, idx, y, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = cpt.distill_topk(z, t, idx, y, **kw)
    for i in range(4):
        z.copy_(z.roll(1, 0))
        y.copy_(y.roll(1, 0))
        want = cpt.distill_topk(z, t, idx, y, **kw)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])


def test_another_stream(device):
    cpt = _cpt()
    z, t, idx, y, _ = _inputs(64, 9000, 5, torch.bfloat16, device)
    want = cpt.distill_topk(z, t, idx, y, alpha=0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cpt.distill_topk(z, t, idx, y, alpha=0.5)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(device):
    cpt = _cpt()
    z = torch.zeros(4, 50, device=device)
    t, i = torch.zeros(4, 3, device=device), torch.zeros(4, 3, dtype=torch.int64, device=device)
    y = torch.zeros(4, dtype=torch.int64, device=device)
    wide = torch.zeros(1, 524289, device=device)
    for bad in (lambda: cpt.distill_topk(z, t, i.short()), lambda: cpt.distill_topk(z, t[:3], i),
                lambda: cpt.distill_topk(z, t[:3], i[:3]),
                lambda: cpt.distill_topk(z, t, i, alpha=0.5),
                lambda: cpt.distill_topk(z, t, i, y[:2]),
                lambda: cpt.distill_topk(z, t, i, y.float()),
                lambda: cpt.distill_topk(z, t, i, temperature=0.0),
                lambda: cpt.distill_topk(z, t, i, reduction="batchmean"),
                lambda: cpt.distill_topk(z, t, i, grad_out=torch.ones(4, device=device)),
                lambda: cpt.distill_topk(z.double(), t, i),
                lambda: cpt.distill_topk(z[:1].expand(4, 50), t, i, inplace=True),
                lambda: cpt.distill_topk(z[:, ::2], t, i, inplace=True),
                lambda: cpt.distill_topk(wide, t[:1], i[:1]),
                lambda: cpt.distill_topk(torch.zeros(1, 5000, device=device),
                                         torch.zeros(1, 2049, device=device),
                                         torch.zeros(1, 2049, dtype=torch.int32, device=device))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError):
        cpt.distill_topk(z.cpu(), t, i)


@pytest.mark.parametrize("k", [1, 19])
@pytest.mark.parametrize("tau", [1.0, 4.0, 8.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_shares_keep_their_digits(device, dtype, tau, k):
    """Entries that hold a small part of both softmaxes: the rest's term and the
    columns' gradient are differences between shares near 1.  With s = sum (p + q)
    over the entries' columns, L the largest |log p|, |log q| there, each share is
    good to (2 L + 200) e of itself, and the loss is of first order in them:
    |error| <= tau^2 (4 L + 400) e s (L + 1).  A column outside the entries has
    tau (p_top - P q_top) q / q_rest."""
    g = torch.Generator().manual_seed(k)
    n, v = 40, 24001
    z = torch.randn(n, v, generator=g).to(dtype)
    t = z.float() * 0.5 + torch.randn(n, v, generator=g)
    top = 0.2 * t[:, 100:100 + k]   # not the largest: the entries' share stays small
    idx = torch.arange(100, 100 + k).expand(n, k).contiguous()
    lse = torch.logsumexp(t.double() / tau, 1).float()
    lq = torch.log_softmax(z.double() / tau, 1)
    lp = top.double() / tau - lse.double()[:, None]
    p, q = lp.exp(), lq[:, 100:100 + k].exp()
    a, b = p.sum(1), q.sum(1)
    assert (a < 0.1).all() and (b < 0.1).all()
    want = tau ** 2 * ((p * (lp - q.log())).sum(1) + (1 - a) * (torch.log1p(-a) - torch.log1p(-b)))
    big = torch.maximum(lp.abs().amax(1), q.log().abs().amax(1))
    bound = tau ** 2 * (4 * big + 400) * E * (a + b) * (big + 1)
    loss, grad = _cpt().distill_topk(z.to(device), top.to(device), idx.to(device),
                                     top_lse=lse.to(device), temperature=tau, alpha=1.0,
                                     reduction="none",
                                     grad_out=torch.full((n,), 2.0 ** 12, device=device))
    assert ((loss.cpu().double() - want).abs() <= bound).all()
    out = torch.ones(v, dtype=torch.bool)
    out[100:100 + k] = False
    cond = (lq - torch.log1p(-b)[:, None]).exp()[:, out]
    exact = 2.0 ** 12 * tau * (a - b)[:, None] * cond
    slack = 2.0 ** 12 * tau * (4 * big + 400 + 200)[:, None] * E * (a + b)[:, None] * cond
    off = (grad.cpu().double()[:, out] - exact).abs()
    assert (off <= UNIT[dtype] * exact.abs() + TINY[dtype] + slack).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [0.5, 1.0, 1.5, 2.0, 8.0])
@pytest.mark.parametrize("value", [-1e9, -2.5e8, 1e9])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_far_values(device, dtype, value, tau, tail):
    """Rows that lie wholly beyond what a base of the exponentials reaches, at the
    temperature or at temperature 1 alone: all one value, or a few steps apart (so
    that exact gradients lie below the smallest normal number, 2^-126, too)."""
    for v in (200, 70001):
        z, t, idx, y, lse = _inputs(4, v, 6, dtype, device, tau=tau, tail=tail)
        y[:] = idx[:, 1]
        z[1] = value
        z[2] = (value + 64.0 * (torch.arange(v, device=device) % 3)).to(dtype)
        want = definition(z, t, idx, y, lse, tau, 0.5, -100, "none", 1.0)
        loss, grad = _cpt().distill_topk(z, t, idx, y, top_lse=lse, temperature=tau, alpha=0.5,
                                         reduction="none")
        assert loss.isfinite().all() and grad.isfinite().all()
        _close(loss, want[0], want[2] + 2.0 ** -23 * want[0].abs(), "loss")
        _close(grad, want[1], UNIT[dtype] * want[1].abs() + want[3] + 2.0 ** -126, "gradient")


@pytest.mark.parametrize("tau", [1.0, 1.5, 2.0])
@pytest.mark.parametrize("value", [-1e9, -2.5e8, "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_values_outside_the_entries(device, dtype, value, tau):
    """With a tail, finite logits far below the entries count as the formula has them
    (q_rest about exp(value / tau)); only -inf leaves nothing.  Bounds as above, with
    the range of the entries and of the rest each by itself: 150 at most; a gradient
    may lie below the smallest normal number."""
    value = torch.finfo(dtype).min if value == "lowest" else value
    n, k, alpha = 4, 6, 0.5
    for v in (200, 70001):
        z, t, idx, y, lse = _inputs(n, v, k, dtype, device, tau=tau, tail=True)
        lse += 0.5
        y[:] = idx[:, 1]
        at = z.gather(1, idx)
        z[1:3] = value
        if value > -1e30:
            z[2] = (value + 64.0 * (torch.arange(v, device=device) % 3)).to(dtype)
        z[1:3] = z[1:3].scatter(1, idx[1:3], at[1:3])
        z[3] -= 5e8 if dtype == torch.float32 else 0   # the whole row, entries and rest
        z64, lp = z.double(), t.double() / tau - lse.double()[:, None]
        lq = torch.log_softmax(z64 / tau, 1)
        p, lqj = lp.exp(), lq.gather(1, idx)
        top = torch.zeros_like(z64).scatter_(1, idx, 1.0) > 0
        lo = torch.logsumexp(lq.masked_fill(top, -math.inf), 1)
        rest = 1 - p.sum(1)
        assert (rest > 0.1).all()
        soft = (p * (lp - lqj)).sum(1) + rest * (rest.log() - lo)
        size = (p * (lp.abs() + lqj.abs() + 1)).sum(1) + rest * (rest.log().abs() + lo.abs() + 1)
        l1 = torch.log_softmax(z64, 1)
        hard = -l1.gather(1, y[:, None])[:, 0]
        loss, grad = _cpt().distill_topk(z, t, idx, y, top_lse=lse, temperature=tau, alpha=alpha,
                                         reduction="none")
        off = (12 * (lse.double().abs() + lp.abs().amax(1)) + 8 + k) * E
        want = alpha * tau ** 2 * soft + (1 - alpha) * hard
        bound = 2.0 ** -23 * want.abs() + (1 - alpha) * 550 * E * (hard + 1) \
            + alpha * tau ** 2 * (550 * E * size + off * (lo.abs() + rest.log().abs() + 2))
        _close(loss, want, bound, "loss")
        # 64 bits do not hold log(v) beside the lowest value: not exp(lq - lo)
        cond = torch.softmax((z64 / tau).masked_fill(top, -math.inf), 1)
        dense = torch.zeros_like(z64).scatter_(1, idx, p)
        hot = torch.zeros_like(z64).scatter_(1, y[:, None], 1.0)
        exact = alpha * tau * (lq.exp() - dense - rest[:, None] * cond) \
            + (1 - alpha) * (l1.exp() - hot)
        terms = tau * (lq.exp() + dense + rest[:, None] * cond) + l1.exp() + hot
        _close(grad, exact, UNIT[dtype] * exact.abs() + 550 * E * terms
               + tau * off[:, None] * (dense + cond + lq.exp()) + 2.0 ** -126, "gradient")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_large_teacher_logits(device, tau, tail):
    """Teacher logits about 32768 (a unit in the last place is 2^-8): log p is rounded
    about 0, not about them.  A difference of two of them is exact or rounded once, so
    log p has an error of (4 |log p| + 8) e; with R the rows' ranges of teacher and
    student and sums of fewer than 60 roundings, the loss has
    tau^2 (4 R + 100) e * its terms, and p_rest = 1 - sum p an error of (4 R + 100) e."""
    g = torch.Generator().manual_seed(11)
    n, v, k = 20, 1000, 40
    z = 2 * torch.randn(n, v, generator=g)
    t = 32768 - torch.randint(0, 2000, (n, k), generator=g) / 256.0
    idx = torch.argsort(torch.rand(n, v, generator=g), 1)[:, :k].contiguous()
    t64, lq = t.double() / tau, torch.log_softmax(z.double() / tau, 1)
    base = torch.logsumexp(t64, 1)
    lse = (base + 0.25).float() if tail else None
    lp = t64 - (lse.double() if tail else base)[:, None]
    p, lqj = lp.exp(), lq.gather(1, idx)
    soft, size = (p * (lp - lqj)).sum(1), (p * (lp.abs() + lqj.abs() + 1)).sum(1)
    err = (4 * (1 + (z.amax(1) - z.amin(1)).double() + 8) + 100) * E
    bound = err * size
    if tail:
        rest = 1 - p.sum(1)
        lo = torch.logsumexp(lq.scatter(1, idx, -math.inf), 1)
        soft = soft + rest * (rest.log() - lo)
        bound = bound + err * (rest.log().abs() + lo.abs() + 2)
    loss, _ = _cpt().distill_topk(z.to(device), t.to(device), idx.to(device),
                                  top_lse=lse.to(device) if tail else None, temperature=tau,
                                  reduction="none", want_grad=False)
    _close(loss.cpu(), tau ** 2 * soft, tau ** 2 * bound + 2.0 ** -23 * tau ** 2 * soft.abs(),
           "loss")


def test_sum_over_the_widest_row(device):
    """A sum of equal exponentials 1 + 2^-15 - 2^-20, which a chain of 1024 of them
    rounds down by half a unit at every other step.  With chains of at most 150 terms,
    the block's exchange (16) and the logarithm's and products' roundings (60 at this
    size), log sum exp - z = log v is off by 230 e at most."""
    v = 524288
    value = math.log(1 + 2.0 ** -15 - 2.0 ** -20)
    z = torch.full((3, v), value, device=device)
    t, idx = torch.zeros(3, 1, device=device), torch.zeros(3, 1, dtype=torch.int64, device=device)
    y = torch.arange(3, device=device)
    loss, _ = _cpt().distill_topk(z, t, idx, y, alpha=0.0, reduction="none", want_grad=False)
    assert ((loss.double() - math.log(v)).abs() <= 230 * E).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [1.0, 1.5, 2.0])
@pytest.mark.parametrize("n,v,dtype", [(7000, 515, torch.bfloat16), (7000, 515, torch.float32),
                                       (2200, 8209, torch.float16), (1100, 8209, torch.float32),
                                       (600, 33001, torch.float32)])
def test_many_rows_a_block(device, n, v, dtype, tau, tail):
    """More rows than blocks: each goes over several, ignored ones between them, with
    entries that occur twice or not at all."""
    z, t, idx, y, lse = _inputs(n, v, 9, dtype, device, tau=tau, tail=tail)
    idx[::5, 1] = idx[::5, 0]
    idx[3::7, 2] = -1
    if tail:
        lse += 0.5
    gout = 4096.0 if dtype == torch.float16 else 1.0
    loss, grad = check(z, t, idx, y, lse, tau, 0.5, reduction="none", gout=gout)
    only, _ = _cpt().distill_topk(z, t, idx, y, top_lse=lse, temperature=tau, alpha=0.5,
                                  reduction="none", want_grad=False)
    want = definition(z, t, idx, y, lse, tau, 0.5, -100, "none", 1.0)
    _close(only, want[0], want[2] + 2.0 ** -23 * want[0].abs(), "loss alone")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("tau", [1.0, 1.5, 2.0, 8.0])
def test_far_values_without_a_gradient(device, tau, tail):
    """Rows that are moved to 0, whose columns are all read again, give the losses that
    the pass with the gradient gives (the same sums in another order)."""
    for v in (200, 70001):
        z, t, idx, y, lse = _inputs(4, v, 6, torch.float32, device, tau=tau, tail=tail)
        y[:] = idx[:, 1]
        at = z.gather(1, idx)
        z[1:3] = -1e9
        z[2] = z[2].scatter(0, idx[2], at[2])
        kw = dict(top_lse=lse, temperature=tau, alpha=0.5, reduction="none")
        with_grad, _ = _cpt().distill_topk(z, t, idx, y, **kw)
        alone, _ = _cpt().distill_topk(z, t, idx, y, want_grad=False, **kw)
        assert alone.isfinite().all()
        assert ((alone - with_grad).abs() <= 2 * 550 * E * (1 + with_grad.abs())).all()
