"""Head norms and position rotation against the formula in 64 bits on the CPU.

Tolerances.  u: half a step of the output's type.  A rotated pair in fp32: the norm's
scale (a sum of D squares in a tree of registers and exchanges, a root, two
products) is good to 16 x 2^-24, cos and sin to 4 x 2^-24 absolute, the products
and the sum to 3 x 2^-24: under 32 x 2^-24 of the pair's length.  The gradient's
head has two such terms and a mean of D products: 64 x 2^-24 of rho (|g w| + |n|
rms(g w)).  A weight's gradient is a sum of N terms each good to 32 x 2^-24: (N + 32)
2^-24 of the sum of their sizes."""

import pytest
import torch

import compact_amd as cpt

pytestmark = pytest.mark.gpu

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _turn(x, pos, inv_freq, inter, scaling=1.0, sign=1.0):
    r = 2 * inv_freq.numel()
    t = pos.double()[..., None, None] * inv_freq.double()
    c, s = scaling * t.cos(), sign * scaling * t.sin()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    pair = [a * c - b * s, b * c + a * s]
    turned = torch.stack(pair, -1).flatten(-2) if inter else torch.cat(pair, -1)
    return torch.cat([turned, x[..., r:]], -1)


def _length(x, r, inter):
    """Each element's pair's length (an element's own size past the rotated ones)."""
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    n = (a * a + b * b).sqrt()
    n = torch.stack([n, n], -1).flatten(-2) if inter else torch.cat([n, n], -1)
    return torch.cat([n, x[..., r:].abs()], -1)


def _make(b, s, h, hk, d, r, dt, norm, seed=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(b, s, h, d, generator=g), torch.randn(b, s, hk, d, generator=g)
    q[..., ::5] *= 10
    pos = torch.randint(0, far, (b, s), generator=g)
    inv = (10000.0 ** (-torch.arange(0, r, 2).double() / r)).float()
    w = [(1 + 0.1 * torch.randn(d, generator=g)).to(dt) if norm else None for _ in range(2)]
    return q.to(dt), k.to(dt), pos, inv, *w


def _want(x, pos, inv, w, inter, scaling=1.0):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
    return _turn(x, pos, inv, inter, scaling), x


def _check(got, x, pos, inv, w, inter, dt, scaling=1.0):
    want, n = _want(x, pos, inv, w, inter, scaling)
    tol = torch.finfo(dt).eps / 2 * want.abs() + \
        32 * 2.0 ** -24 * max(1, scaling) * _length(n, 2 * inv.numel(), inter)
    tol += torch.finfo(dt).tiny * torch.finfo(dt).eps
    bad = ((got.cpu().double() - want).abs() > tol).sum()
    assert bad == 0, f"{bad} of {want.numel()}"


SHAPES = [(1, 1, 1, 1, 2, 2), (4, 1, 32, 4, 64, 64), (2, 33, 6, 2, 128, 128), (3, 7, 5, 3, 80, 40),
          (2, 5, 3, 1, 96, 96), (1, 9, 2, 2, 6, 4), (2, 3, 7, 1, 20, 20), (1, 130, 3, 2, 48, 16),
          (1, 2, 2, 1, 1024, 1024), (2, 3, 2, 2, 258, 130), (1, 1500, 2, 1, 16, 16),
          (2, 5, 3, 1, 42, 42), (1, 4, 2, 1, 300, 150), (1, 3, 2, 1, 1024, 510), (1, 3, 2, 1, 1022, 510),
          (2, 3, 1, 1, 18, 16), (1, 70, 1, 1, 128, 128)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(device, dtype, norm, inter, shape):
    dt = TYPES[dtype]
    q, k, pos, inv, wq, wk = _make(*shape, dt, norm)
    on = [None if t is None else t.to(device) for t in (q, k, pos, inv, wq, wk)]
    gq, gk = cpt.qk_rope(*on[:4], w_q=on[4], w_k=on[5], eps=EPS, interleaved=inter)
    assert gq.is_contiguous() and gq.dtype == dt
    _check(gq, q, pos, inv, wq, inter, dt)
    _check(gk, k, pos, inv, wk, inter, dt)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(device, dtype, inter, shape):
    dt = TYPES[dtype]
    q, k, pos, inv, wq, wk = _make(*shape, dt, True, seed=1)
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g).to(dt) for t in (q, k))
    on = [t.to(device) for t in (dq, dk, q, k, pos, inv, wq, wk)]
    got = cpt.qk_rope_backward(*on[:6], w_q=on[6], w_k=on[7], eps=EPS, interleaved=inter)
    u = torch.finfo(dt).eps / 2
    for d, x, w, gx, gw in ((dq, q, wq, got[0], got[2]), (dk, k, wk, got[1], got[3])):
        dn = _turn(d.double(), pos, inv, inter, sign=-1.0)
        x = x.double()
        rho = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n, gw_ = x * rho, dn * w.double()
        want = rho * (gw_ - n * (gw_ * n).mean(-1, keepdim=True))
        size = _length(dn, 2 * inv.numel(), inter) * w.double().abs()
        tol = u * want.abs() + 64 * 2.0 ** -24 * rho * (
            size + n.abs() * gw_.square().mean(-1, keepdim=True).sqrt())
        tol += torch.finfo(dt).tiny * torch.finfo(dt).eps
        assert ((gx.cpu().double() - want).abs() <= tol).all()
        terms = dn * n
        want_w = terms.sum((0, 1, 2))
        sizes = (_length(dn, 2 * inv.numel(), inter) * n.abs()).sum((0, 1, 2))
        tol = u * want_w.abs() + (terms[..., 0].numel() + 32) * 2.0 ** -24 * sizes
        assert ((gw.cpu().double() - want_w).abs() <= tol).all()


def test_far_positions(device):
    """A position in the millions turns as exactly as a near one, int32 and int64."""
    q, k, _, inv, _, _ = _make(1, 6, 2, 1, 64, 64, torch.float32, False)
    for pos in ([0, 1, 999999, 12345678, 2 ** 31 - 1, -7], [2 ** 33 + 5, 2 ** 35, 1, 2, 3, -2 ** 31]):
        pos = torch.tensor(pos)
        for p in (pos, pos.int()) if pos.abs().max() < 2 ** 31 else (pos,):
            gq, gk = cpt.qk_rope(q.to(device), k.to(device), p.to(device), inv.to(device))
            _check(gq, q, pos, inv, None, False, torch.float32)
            _check(gk, k, pos, inv, None, False, torch.float32)


def test_layouts_positions_and_scaling(device):
    """Views of one projection, heads before tokens, three axes, no positions."""
    dt = torch.bfloat16
    q, k, pos, inv, wq, wk = _make(3, 11, 4, 2, 64, 64, dt, True, seed=3)
    qkv = torch.cat([q, k, k], 2).to(device)
    kw = dict(w_q=wq.to(device), w_k=wk.to(device), eps=EPS)
    inv_d = inv.to(device)
    want = cpt.qk_rope(q.to(device), k.to(device), pos.to(device), inv_d, **kw)
    got = cpt.qk_rope(qkv[:, :, :4], qkv[:, :, 4:6], pos.to(device), inv_d, **kw)
    first = [t.to(device).transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    got2 = cpt.qk_rope(*first, pos.to(device), inv_d, **kw)
    wide = torch.zeros(3, 11, 6, 99, dtype=dt, device=device)     # odd strides: unaligned rows
    wide[..., 3:67] = torch.cat([q, k], 2).to(device)
    got3 = cpt.qk_rope(wide[:, :, :4, 3:67], wide[:, :, 4:, 3:67], pos.to(device), inv_d, **kw)
    for g in (got, got2, got3):
        assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1])
    one = [cpt.qk_rope(q[i].to(device), k[i].to(device), pos[i].to(device), inv_d, **kw)
           for i in range(3)]
    assert torch.equal(torch.stack([o[0] for o in one]), want[0])
    row = torch.arange(11, device=device)
    a = cpt.qk_rope(q.to(device), k.to(device), None, inv_d, **kw)
    for p in (row, row[None], row.expand(3, 11)):
        b = cpt.qk_rope(q.to(device), k.to(device), p, inv_d, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    got = cpt.qk_rope(q.to(device), k.to(device), pos.to(device), inv_d, scaling=1.25)
    _check(got[0], q, pos, inv, None, False, dt, 1.25)
    w32 = dict(w_q=wq.float().to(device), w_k=wk.float().to(device), eps=EPS)
    got = cpt.qk_rope(q.to(device), k.to(device), pos.to(device), inv_d, **w32)
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("norm", [False, True])
def test_inplace(device, norm):
    q, k, pos, inv, wq, wk = (None if t is None else t.to(device) for t in
                              _make(2, 37, 6, 2, 96, 64, torch.bfloat16, norm, seed=5))
    kw = dict(w_q=wq, w_k=wk, eps=EPS)
    want = cpt.qk_rope(q, k, pos, inv, **kw)
    qkv = torch.cat([q, k, k], 2)
    old = qkv.clone()
    a, b = qkv[:, :, :6], qkv[:, :, 6:8]
    got = cpt.qk_rope(a, b, pos, inv, inplace=True, **kw)
    assert got[0] is a and got[1] is b
    assert torch.equal(qkv[:, :, :6], want[0]) and torch.equal(qkv[:, :, 6:8], want[1])
    assert torch.equal(qkv[:, :, 8:], old[:, :, 8:])


@pytest.mark.parametrize("d,r", [(64, 32), (10, 4)])
@pytest.mark.parametrize("inter", [False, True])
def test_infinities_past_the_rotated_columns(device, d, r, inter):
    """Without norms a column that does not turn is itself, whatever the others are."""
    q, k, pos, inv, _, _ = _make(1, 3, 2, 1, d, r, torch.float32, False)
    q[0, 1, 0, r + 1] = float("inf")
    q[0, 1, 1, d - 1] = float("nan")
    q[0, 2, 0, r] = -float("inf")
    for back in (False, True):
        got, _ = cpt.qk_rope(*(t.to(device) for t in (q, k, pos, inv)), interleaved=inter,
                             inverse=back)
        assert torch.equal(got[..., r:].cpu().nan_to_num(7.0), q[..., r:].nan_to_num(7.0))
        assert got[..., :r].isfinite().all()


def test_zeros_nan_and_empty(device):
    """A head of zeros stays zeros; NaN and inf stay in their head; no tokens, no launch."""
    q, k, pos, inv, wq, wk = (t.to(device) for t in
                              _make(1, 4, 3, 1, 32, 32, torch.float32, True))
    q[0, 1] = 0
    q[0, 2, 1, 5] = float("nan")
    q[0, 3, 0, 7] = float("inf")
    gq, _ = cpt.qk_rope(q, k, pos, inv, w_q=wq, w_k=wk)
    assert (gq[0, 1] == 0).all()
    bad = torch.zeros(4, 3, dtype=torch.bool, device=device)
    bad[2, 1] = bad[3, 0] = True
    assert torch.equal(~gq[0].isfinite().all(-1), bad)
    d = torch.ones_like(q)
    dq, _, dw, _ = cpt.qk_rope_backward(d[:, :2], torch.ones_like(k)[:, :2], q[:, :2], k[:, :2],
                                        pos[:, :2], inv, w_q=wq, w_k=wk)
    assert dq.isfinite().all() and dw.isfinite().all()
    none = cpt.qk_rope(q[:, :0], k[:, :0], pos[:, :0], inv, w_q=wq, w_k=wk)
    assert none[0].shape == (1, 0, 3, 32)
    grads = cpt.qk_rope_backward(d[:, :0], k[:, :0], q[:, :0], k[:, :0], pos[:, :0], inv, w_q=wq,
                                 w_k=wk)
    assert grads[0].numel() == 0 and (grads[2] == 0).all()


@pytest.mark.parametrize("norm", [False, True])
def test_function_against_autograd(device, norm):
    """Gradients of the Function and module against autograd of the formula and against
    differences, in fp32."""
    q, k, pos, inv, wq, wk = _make(2, 6, 3, 2, 24, 16, torch.float32, norm, seed=7)
    m = cpt.QKNormRope(24, rotary=16, norm=norm, eps=EPS, device=device)
    assert torch.equal(m.inv_freq.cpu(), inv)
    if norm:
        with torch.no_grad():
            m.w_q.copy_(wq)
            m.w_k.copy_(wk)
    a, b = (t.to(device).requires_grad_(True) for t in (q, k))
    g = torch.Generator().manual_seed(2)
    gq, gk = (torch.randn(t.shape, generator=g) for t in (q, k))
    oq, ok = m(a, b, pos.to(device))
    ((oq * gq.to(device)).sum() + (ok * gk.to(device)).sum()).backward()
    p = [t.double().requires_grad_(True) for t in (q, k)]
    w = [t.double().requires_grad_(True) if norm else None for t in (wq, wk)]
    loss = sum((_want(x, pos, inv, y, False)[0] * z.double()).sum()
               for x, y, z in zip(p, w, (gq, gk)))
    loss.backward()
    pairs = [(a.grad, p[0].grad), (b.grad, p[1].grad)]
    if norm:
        pairs += [(m.w_q.grad, w[0].grad), (m.w_k.grad, w[1].grad)]
    for got, want in pairs:
        # 64 x 2^-24 of terms as large as the gradient's largest
        assert (got.cpu().double() - want).abs().max() <= 2.0 ** -17 * want.abs().max()

    def value(x):
        return (_want(x, pos, inv, wq, False)[0] * gq.double()).sum()

    step = torch.zeros_like(q).double()
    step[1, 2, 1] = torch.randn(24, generator=g).double()
    # third derivatives times 1e-4 squared are under 1e-6 of the slope here
    slope = (value(q.double() + 1e-4 * step) - value(q.double() - 1e-4 * step)) / 2e-4
    assert abs((a.grad.cpu().double() * step).sum() - slope) <= 1e-5 * (1 + abs(slope))


def test_differentiable_once_and_casts(device):
    m = cpt.QKNormRope(16, device=device)
    q = torch.randn(1, 3, 2, 16, device=device, requires_grad=True)
    k = torch.randn(1, 3, 1, 16, device=device)
    oq, _ = m(q, k)
    g, = torch.autograd.grad(oq.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    freq = m.inv_freq.clone()
    m.to(torch.bfloat16)
    assert m.inv_freq.dtype == torch.float32 and torch.equal(m.inv_freq, freq)
    assert m.w_q.dtype == torch.bfloat16 and "inv_freq" not in m.state_dict()


def test_gradients_as_attention_leaves_them(device):
    """Expanded gradients and those with heads before tokens; float32 weights."""
    q, k, pos, inv, wq, wk = (t.to(device) for t in
                              _make(2, 9, 4, 2, 64, 32, torch.bfloat16, True, seed=6))
    wq, wk = wq.float(), wk.float()
    d = [torch.randn(t.shape, device=device).bfloat16() for t in (q, k)]
    kw = dict(w_q=wq, w_k=wk, eps=EPS)
    want = cpt.qk_rope_backward(*d, q, k, pos, inv, **kw)
    assert want[2].dtype == torch.float32
    first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in d]
    got = cpt.qk_rope_backward(*first, q, k, pos, inv, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = torch.ones((), device=device, dtype=torch.bfloat16)
    got = cpt.qk_rope_backward(one.expand_as(q), one.expand_as(k), q, k, pos, inv, **kw)
    want = cpt.qk_rope_backward(torch.ones_like(q), torch.ones_like(k), q, k, pos, inv, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = cpt.qk_rope_backward(one.expand_as(q), one.expand_as(k), None, None, pos, inv)
    want = cpt.qk_rope(torch.ones_like(q), torch.ones_like(k), pos, inv, inverse=True)
    assert torch.equal(none[0], want[0]) and none[2] is None


def test_repeats_bits_streams_and_graph(device):
    """The same bits on every run, on another stream, and in a graph replayed with other
    work between."""
    q, k, pos, inv, wq, wk = (t.to(device) for t in
                              _make(4, 300, 8, 2, 128, 128, torch.bfloat16, True, seed=4))
    d = [torch.randn_like(q), torch.randn_like(k)]

    def both():
        f = cpt.qk_rope(q, k, pos, inv, w_q=wq, w_k=wk)
        return (*f, *cpt.qk_rope_backward(*d, q, k, pos, inv, w_q=wq, w_k=wk))

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
    for i in range(3):
        q.mul_(-1 if i else 1)
        graph.replay()
        again = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_offsets_past_32_bits(device):
    """Tokens that start past 2^31 elements: as a call of their own."""
    s, h, d = 131100, 128, 128
    q = torch.zeros(1, s, h, d, dtype=torch.bfloat16, device=device)
    k = torch.randn(1, s, 1, d, device=device).bfloat16()
    _, _, _, inv, wq, wk = (t.to(device) for t in _make(1, 1, 1, 1, d, d, torch.bfloat16, True))
    g = torch.Generator(device).manual_seed(1)
    q[:, -3:] = torch.randn(1, 3, h, d, device=device, generator=g).bfloat16()
    pos = torch.arange(s, device=device)
    kw = dict(w_q=wq, w_k=wk, eps=EPS)
    big, _ = cpt.qk_rope(q, k, None, inv, **kw)
    small, _ = cpt.qk_rope(q[:, -3:], k[:, -3:], pos[-3:], inv, **kw)
    assert torch.equal(big[:, -3:], small) and (big[:, :7] == 0).all()
    dq, *_ = cpt.qk_rope_backward(q, k, q, k, pos, inv, **kw)
    small, *_ = cpt.qk_rope_backward(q[:, -3:], k[:, -3:], q[:, -3:], k[:, -3:], pos[-3:], inv, **kw)
    assert torch.equal(dq[:, -3:], small)


def test_inference_mode(device):
    with torch.inference_mode():
        q, k, pos, inv, _, _ = (t if t is None else t.to(device) for t in
                                _make(4, 1, 4, 2, 64, 64, torch.float16, False))
        want = cpt.qk_rope(q, k, pos, inv)
        got = cpt.qk_rope(q, k, pos, inv, inplace=True)
        assert torch.equal(got[0], want[0]) and torch.equal(k, want[1])
