"""Token log probabilities, entropy and alternatives against the formulas in 64 bits.

Tolerances.  With t = (x - max) / T: an exponential is good to (3 + |t|) 2^-23, a
thread adds a chain of V / 256 of them at most (and 20 in the joins), so log s is
good to (V / 256 + 26 + 2 H) 2^-24 x 1 (weights p make |t| the entropy), a log
probability adds 4 |log p| 2^-24, the entropy a second sum of that kind.  lse adds
its own rounding.  The gradient: p good to (V / 256 + 32 + 4 |log p|) 2^-24, and half
a step of its type.  Alternatives are whole numbers: equal."""

import pytest
import torch

import compact_amd as cpt

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24


def _logits(rows, vocab, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = 2 * torch.randn(rows, vocab, generator=g)
    at = torch.randint(0, vocab, (rows, min(24, vocab)), generator=g)
    z.scatter_add_(1, at, 4 + 8 * torch.rand(at.shape, generator=g))
    y = at[:, 0].clone()
    return z.to(dt), y


def _order(z, k):
    """Columns of the k largest values of each row, equals by column, NaN largest."""
    return torch.sort(z.double(), dim=1, descending=True, stable=True).indices[:, :k]


def _check(r, z, y, tau, k, live=None):
    v = z.shape[1]
    t = z.double() / tau
    lp = torch.log_softmax(t, 1)
    h = torch.special.entr(lp.exp()).sum(1)
    base = (v / 256 + 26 + 2 * h) * U
    live = torch.ones(len(z), dtype=torch.bool) if live is None else live

    def close(got, want, tol):
        got = got.cpu().double()
        assert (got[~live] == 0).all()
        assert ((got - want).abs() <= tol)[live].all(), float((got - want).abs()[live].max())

    want = lp.gather(1, y.clamp(0, v - 1)[:, None])[:, 0]
    close(r.logprobs, want, base + 4 * want.abs() * U)
    close(r.entropy, h, 2 * base * (1 + h))
    lse = torch.logsumexp(t, 1)
    close(r.lse, lse, base + 3 * U * (lse.abs() + t.amax(1).abs()))
    if k:
        idx = _order(z, k)
        idx[~live] = -1
        assert torch.equal(r.top_indices.cpu(), idx)
        want = lp.gather(1, idx.clamp(min=0))
        got = r.top_logprobs.cpu().double()
        assert (got[~live] == -float("inf")).all()
        ok = (got - want).abs() <= base[:, None] + 4 * want.abs() * U
        assert (ok | (got == want))[live].all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,k,tau", [
    (1, 1, 1, 1.0), (3, 5, 5, 0.7), (5, 100, 20, 1.0), (2, 511, 128, 1.3), (4, 512, 64, 1.0),
    (3, 1000, 128, 1.0), (2, 2047, 17, 1.0), (2, 4097, 1, 0.7), (7, 32000, 5, 1.0),
    (2, 50021, 50, 1.3), (1, 131075, 128, 1.0), (600, 5003, 20, 1.0),
    (257, 70001, 30, 0.7), (300, 9000, 128, 1.0), (300, 9000, 48, 1.0),
    (300, 12345, 0, 1.0), (1000, 16384, 20, 1.0), (520, 2048, 0, 1.0)])
def test_forward(device, dtype, rows, vocab, k, tau):
    z, y = _logits(rows, vocab, TYPES[dtype], seed=vocab)
    r = cpt.token_logprobs(z.to(device), y.to(device), temperature=tau, top_k=k)
    _check(r, z, y, tau, k)
    assert (r.top_indices is None) == (k == 0)


@pytest.mark.parametrize("rows", [3, 700])
def test_rows_left_out(device, rows):
    z, y = _logits(rows, 3001, torch.bfloat16, seed=1)
    y[0], y[1], y[2] = -100, 3001, -1
    live = torch.ones(rows, dtype=torch.bool)
    live[:3] = False
    for t in (y, y.int()):
        _check(cpt.token_logprobs(z.to(device), t.to(device), top_k=7), z, y, 1.0, 7, live)
    r = cpt.token_logprobs(z.to(device), None, top_k=7)
    assert r.logprobs is None
    assert torch.equal(r.top_indices.cpu(), _order(z, 7))
    kept = cpt.token_logprobs(z.to(device), y.to(device), ignore_index=int(y[-1]), top_k=2)
    assert (kept.top_indices[y.to(device) == y[-1]] == -1).all()


@pytest.mark.parametrize("vocab", [40, 900, 20000])
@pytest.mark.parametrize("rows", [1, 800])
def test_ties_masks_and_nan(device, vocab, rows):
    """Constant rows, rows with few finite logits, with none, at the type's lowest, in
    rising and falling order, and with NaN and infinities."""
    k, inf = 20, float("inf")
    low = torch.finfo(torch.float32).min
    z = torch.randn(11, vocab, generator=torch.Generator().manual_seed(3))
    z[0] = 0.25
    z[1] = -inf
    z[1, 5], z[1, 7] = 1.0, 1.0
    z[2] = -inf
    z[3] = low
    z[4, 3:] = low
    z[5] = torch.arange(vocab).float() * 0.01
    z[6] = -torch.arange(vocab).float() * 0.01
    z[7] = (torch.arange(vocab) % 3).float()
    z[8, 11] = z[8, 31] = float("nan")
    z[9, 12] = inf
    z[10] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)
    y = torch.tensor([1, 5, 2, 9, 1, 4, 0, 2, 3, 12, 5])
    n = rows if rows > 11 else 11
    z, y = z.repeat(-(-n // 11), 1)[:n], y.repeat(-(-n // 11))[:n]
    r = cpt.token_logprobs(z.to(device), y.to(device), top_k=k)
    got = [None if t is None else t.cpu() for t in r]
    for i in range(min(n, 22)):
        kind = i % 11
        assert torch.equal(got[4][i], _order(z[i:i + 1], k)[0]), kind
        if kind == 2:
            assert got[0][i] == -inf and got[1][i] == 0 and got[2][i] == -inf
            assert (got[3][i] == -inf).all()
        elif kind in (8, 9):
            assert got[0][i].isnan() and got[1][i].isnan() and got[3][i].isnan().all()
        else:
            one = cpt.TokenLogprobs(*[None if t is None else t[i:i + 1] for t in r[:5]], None)
            _check(one, z[i:i + 1], y[i:i + 1], 1.0, k)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,tau", [(1, 1, 1.0), (3, 7, 0.7), (5, 1001, 1.0),
                                            (2, 8192, 1.3), (9, 32003, 1.0), (300, 515, 0.7)])
@pytest.mark.parametrize("which", ["both", "logprobs", "entropy"])
def test_backward(device, dtype, rows, vocab, tau, which):
    dt = TYPES[dtype]
    z, y = _logits(rows, vocab, dt, seed=vocab + 1)
    if rows > 2:
        y[1] = -100
    g = torch.Generator().manual_seed(5)
    a = torch.randn(rows, generator=g) if which != "entropy" else None
    b = torch.randn(rows, generator=g) if which != "logprobs" else None
    zd = z.to(device)
    r = cpt.token_logprobs(zd, y.to(device), temperature=tau, stats=True)
    on = [None if t is None else t.to(device) for t in (a, b)]
    got = cpt.token_logprobs_backward(zd, y.to(device), r.lse, r.entropy, *on, stats=r.stats,
                                      temperature=tau)
    a = torch.zeros(rows) if a is None else a
    b = torch.zeros(rows) if b is None else b
    x = z.double().requires_grad_(True)
    lp = torch.log_softmax(x / tau, 1)
    live = (y >= 0).double()
    h = -(lp.exp() * lp).sum(1)
    (live * (a * lp.gather(1, y.clamp(min=0)[:, None])[:, 0] + b * h)).sum().backward()
    lp, h = lp.detach(), h.detach()
    rel = (vocab / 256 + 32 + 4 * lp.abs()) * U
    hot = torch.zeros_like(lp).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    size = a.abs()[:, None] * (hot + lp.exp()) + \
        b.abs()[:, None] * lp.exp() * (1 + lp.abs() + h[:, None])
    tol = torch.finfo(dt).eps / 2 * x.grad.abs() + rel * size / tau
    tol += torch.finfo(dt).tiny * torch.finfo(dt).eps
    assert ((got.cpu().double() - x.grad).abs() <= tol).all()
    # lse in stats' place: one rounding of it more
    if which == "both":
        other = cpt.token_logprobs_backward(zd, y.to(device), r.lse, r.entropy, *on,
                                            temperature=tau)
        tol += U * r.lse.cpu().double().abs()[:, None] * size / tau * 2
        tol += 4 * U * (z.double() / tau).abs() * size / tau
        assert ((other.cpu().double() - x.grad).abs() <= tol).all()


def test_backward_of_masked_rows(device):
    """-inf columns get zero, a row of nothing else zeros, logits in the thousands and rows
    at the type's lowest their softmax."""
    inf, low = float("inf"), torch.finfo(torch.float32).min
    z = torch.randn(5, 1000, generator=torch.Generator().manual_seed(8))
    z[0, ::2] = -inf
    z[1] = -inf
    z[2] += 5e4
    z[3] = low
    z[4, 10:] = low
    y = torch.tensor([1, 1, 4, 3, 2])
    x = z.to(device).requires_grad_(True)
    r = cpt.token_scores(x, y.to(device))
    (r[0].sum() + 0.5 * r[1].sum()).backward()
    got = x.grad.cpu().double()
    assert (got[0, ::2] == 0).all() and (got[1] == 0).all() and got.isfinite().all()
    for i in (0, 2, 3, 4):
        keep = z[i] > -inf
        t = z[i][keep].double()
        t = (t - t.max()).requires_grad_(True)
        lp = torch.log_softmax(t, 0)
        hit = int(keep[:y[i]].sum())
        (lp[hit] - 0.5 * (lp.exp() * lp).sum()).backward()
        # 36 x 2^-24 of terms up to 1.5 (1 + |log p|)
        assert (got[i][keep] - t.grad).abs().max() <= 100 * U


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_logits_and_inplace(device, dtype):
    z, y = _logits(30, 777, TYPES[dtype], seed=6)
    z, y = z.view(5, 6, 777).to(device), y.view(5, 6).to(device)
    view, labels = z[:, :-1], y[:, 1:]
    want = cpt.token_logprobs(view.contiguous(), labels.contiguous(), top_k=3, stats=True)
    got = cpt.token_logprobs(view, labels, top_k=3, stats=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    d = torch.randn(5, 5, device=device)
    grad = cpt.token_logprobs_backward(view, labels, None, got.entropy, d, d, stats=got.stats)
    assert grad.is_contiguous()
    last = z[:, -1].clone()
    same = cpt.token_logprobs_backward(view, labels, None, got.entropy, d, d, stats=got.stats,
                                       inplace=True)
    assert same is view and torch.equal(view, grad) and torch.equal(z[:, -1], last)


def test_function(device):
    """The Function's gradient against differences; in place; graphs that still need the
    logits refuse; once differentiable."""
    z, y = _logits(4, 300, torch.float32, seed=2)
    x = z.to(device).requires_grad_(True)
    lp, h, lse, tp, ti = cpt.token_scores(x, y.to(device), temperature=0.8, top_k=4)
    assert not lse.requires_grad and not tp.requires_grad
    (lp.sum() - 0.3 * h.sum()).backward()

    def value(t):
        q = torch.log_softmax(t / 0.8, 1)
        return (q.gather(1, y[:, None]).sum() + 0.3 * (q.exp() * q).sum())

    step = torch.randn(z.shape, generator=torch.Generator().manual_seed(1)).double()
    slope = (value(z.double() + 1e-5 * step) - value(z.double() - 1e-5 * step)) / 2e-5
    # the sum of 1200 entries each good to 40 x 2^-24 of terms up to 2; differences to 1e-8
    assert abs((x.grad.cpu().double() * step).sum() - slope) <= 1e-4

    leaf = z.to(device).requires_grad_(True)
    mid = leaf * 1.0
    cpt.token_scores(mid, y.to(device), temperature=0.8, inplace=True)[0].sum().backward()
    ref = z.to(device).requires_grad_(True)
    cpt.token_scores(ref, y.to(device), temperature=0.8)[0].sum().backward()
    assert torch.equal(leaf.grad, ref.grad)
    mid = leaf * 1.0
    lp = cpt.token_scores(mid, y.to(device), inplace=True)[0].sum()
    lp.backward(retain_graph=True)
    with pytest.raises(RuntimeError):       # the logits are gone
        lp.backward()
    with pytest.raises(RuntimeError):       # a leaf's gradient would be the leaf
        cpt.token_scores(leaf, y.to(device), inplace=True)
    with torch.no_grad():                   # no gradient: nothing to refuse
        cpt.token_scores(leaf, y.to(device), inplace=True)
    leaf = z.to(device).requires_grad_(True)
    mid = leaf.exp()        # its gradient needs mid itself
    lp = cpt.token_scores(mid, y.to(device), inplace=True)[0]
    with pytest.raises(RuntimeError):
        lp.sum().backward()
    leaf = z.to(device).requires_grad_(True)
    lp = cpt.token_scores(leaf, y.to(device))[0]
    g, = torch.autograd.grad(lp.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    none = cpt.token_scores(leaf, None)
    assert none[0] is None
    none[1].sum().backward()
    assert leaf.grad.abs().max() > 0


def test_empty_streams_and_graph(device):
    r = cpt.token_logprobs(torch.empty(0, 50, device=device),
                           torch.empty(0, dtype=torch.long, device=device), top_k=2)
    assert r.logprobs.shape == (0,) and r.top_indices.shape == (0, 2)
    z, y = (t.to(device) for t in _logits(900, 9001, torch.bfloat16, seed=4))
    d = torch.randn(900, device=device)

    def both():
        r = cpt.token_logprobs(z, y, top_k=9, stats=True)
        return (*r, cpt.token_logprobs_backward(z, y, None, r.entropy, d, d, stats=r.stats))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(3):
        z.mul_(0.75)
        graph.replay()
        again = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_offsets_past_32_bits(device):
    """Rows that start past 2^31 elements, in both directions."""
    n, v = 67200, 32000
    z = torch.zeros(n, v, dtype=torch.bfloat16, device=device)
    last, y3 = _logits(3, v, torch.bfloat16, seed=9)
    z[-3:] = last.to(device)
    y = torch.full((n,), -100, device=device)
    y[-3:] = y3.to(device)
    r = cpt.token_logprobs(z, y, top_k=5, stats=True)
    tail = cpt.TokenLogprobs(*[t[-3:] for t in r[:5]], None)
    _check(tail, last, y3, 1.0, 5)
    assert (r.top_indices[:-3] == -1).all() and (r.logprobs[:-3] == 0).all()
    d = torch.randn(n, device=device)
    grad = cpt.token_logprobs_backward(z, y, None, r.entropy, d, d, stats=r.stats)
    want = cpt.token_logprobs_backward(z[-3:], y[-3:], None, r.entropy[-3:], d[-3:], d[-3:],
                                       stats=r.stats[:, -3:].contiguous())
    assert torch.equal(grad[-3:], want) and not grad[:-3].any()
