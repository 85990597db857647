"""The residual norm and its gradient against their definitions in 64 bits.

With e = 2^-24 and u one unit in the output type's last place, an fp32 row sum has
chains of at most 16 + 6 + 16 terms, and each value passes fewer than 16 other
operations, so
  residual_out, x   u |exact| + 64 e * (their terms' absolute values)
  dr, dy            u |exact| + 256 e * (likewise, means of absolute values included)
  weights' sums     u |exact| + (rows + 256) e * sum of absolute terms
(the backward takes residual_out and stats as inputs, so their rounding is no
part of its error).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}
E = 2.0 ** -24
EPS = 1e-5

SHAPES = [(1, 1, 1), (1, 1, 4096), (2, 3, 64), (5, 7, 100), (3, 11, 1999), (2, 40, 2048),
          (1, 9, 4097), (2, 2, 8192), (1, 3, 8200), (1, 2, 16384), (70, 1, 40), (1, 1500, 24)]


def _cpt():
    import compact_amd
    return compact_amd


def _gate(kind, shape, gen, dtype):
    s = {"none": None, "channel": shape[-1:], "sequence": (shape[0], 1, shape[2]),
         "token": (*shape[:-1], 1)}[kind]
    return None if s is None else torch.randn(*s, generator=gen).to(dtype)


def _inputs(shape, dtype, wdt, gate, post, device, seed=0):
    g = torch.Generator().manual_seed(seed + shape[-1])
    res, y, dro, dx = (torch.randn(*shape, generator=g).to(dtype) for _ in range(4))
    res[..., 0] *= 30
    w_pre, w_post = ((1 + 0.3 * torch.randn(shape[-1], generator=g)).to(wdt) for _ in range(2))
    ts = (res, y, dro, dx, w_pre, w_post if post else None, _gate(gate, shape, g, wdt))
    return tuple(None if t is None else t.to(device) for t in ts)


def _close(got, exact, slack, what):
    bound = UNIT[got.dtype] * exact.abs() + TINY[got.dtype] + slack
    bad = ~((got.double() - exact).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off by up to " \
        f"{float(((got.double() - exact).abs() / bound)[bad].max()):.2f} bounds"


def _d(t):
    return None if t is None else t.double()


def check_forward(out, res, y, w_pre, w_post, gate, scale, beta, eps):
    """Compares (residual_out, x, stats) with the definition."""
    r64, y64, wp, wq, g = (_d(t) for t in (res, y, w_pre, w_post, gate))
    rho1 = torch.ones_like(y64[..., :1])
    u = y64
    if wq is not None:
        rho1 = (y64.square().mean(-1, keepdim=True) + eps).rsqrt()
        u = y64 * rho1 * wq
    add = scale * (u if g is None else g * u)
    r = beta * r64 + add
    terms = (beta * r64).abs() + add.abs()
    rho2 = torch.ones_like(rho1)
    if wp is not None:
        rho2 = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
        # an error of r moves the row's root mean square by at most its own
        moved = terms.square().mean(-1, keepdim=True).sqrt() * rho2
        _close(out[1], r * rho2 * wp,
               64 * E * ((terms * rho2 * wp).abs() + (r * rho2 * wp).abs() * (1 + moved)), "x")
    _close(out[0], r, 64 * E * terms, "residual_out")
    n = rho1.numel()
    assert torch.allclose(out[2][0].double(), rho1.reshape(n), rtol=64 * E, atol=0)
    want = rho2.reshape(n)
    tol = 64 * E * (1 + (terms.square().mean(-1).sqrt().reshape(n) * want))
    assert ((out[2][1].double() - want).abs() <= tol * want).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(device, dtype, gate, shape):
    cpt = _cpt()
    for post in (True, False):
        res, y, _, _, w_pre, w_post, g = _inputs(shape, dtype, dtype, gate, post, device)
        out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, scale=0.7,
                                residual_scale=1.25, eps=EPS)
        assert out[0].shape == out[1].shape == shape and out[1].dtype == dtype
        check_forward(out, res, y, w_pre, w_post, g, 0.7, 1.25, EPS)


def check_backward(out, dro, dx, ro, y, stats, w_pre, w_post, gate, scale, beta):
    d = ro.shape[-1]
    shape = ro.shape
    dro64, dx64, r, y64, wp, wq, g = (_d(t) for t in (dro, dx, ro, y, w_pre, w_post, gate))
    dro64 = torch.zeros_like(r) if dro64 is None else dro64
    rho1 = stats[0].double().view(*shape[:-1], 1)
    rho2 = stats[1].double().view(*shape[:-1], 1)
    t, size = dro64, dro64.abs()
    if wp is not None:
        n2, v = r * rho2, dx64 * wp
        t = t + rho2 * (v - n2 * (v * n2).mean(-1, keepdim=True))
        size = size + rho2 * (v.abs() + n2.abs() * (v * n2).abs().mean(-1, keepdim=True))
        lead = tuple(range(r.dim() - 1))
        _close(out[2], (dx64 * n2).sum(lead),
               (r.numel() // d + 256) * E * (dx64 * n2).abs().sum(lead), "d_w_pre")
    _close(out[0], beta * t, 256 * E * abs(beta) * size, "d_residual")
    if y is None:
        return
    gg = torch.ones_like(y64[..., :1]) if g is None else g
    n1 = y64 * rho1
    w = wq if wq is not None else torch.ones(d, dtype=torch.float64, device=r.device)
    a, asize = scale * gg * t * w, (scale * gg * w).abs() * size
    dy, ysize = a, asize
    if wq is not None:
        dy = rho1 * (a - n1 * (a * n1).mean(-1, keepdim=True))
        ysize = rho1 * (asize + n1.abs() * (asize * n1.abs()).mean(-1, keepdim=True))
        lead = tuple(range(r.dim() - 1))
        _close(out[3], (scale * gg * t * n1).sum(lead),
               (r.numel() // d + 256) * E * ((scale * gg * n1).abs() * size).sum(lead), "d_w_post")
    _close(out[1], dy, 256 * E * ysize, "d_y")
    if g is not None:
        full, fsize = scale * t * n1 * w, (scale * n1 * w).abs() * size
        axes = [i for i in range(r.dim()) if i - r.dim() + g.dim() < 0
                or g.shape[i - r.dim() + g.dim()] == 1]
        k = 1
        for i in axes:
            k *= shape[i]
        if axes:
            full, fsize = full.sum(axes, keepdim=True), fsize.sum(axes, keepdim=True)
        _close(out[4], full.reshape(g.shape), (k + 256) * E * fsize.reshape(g.shape), "d_gate")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(device, dtype, gate, shape):
    cpt = _cpt()
    for post in (True, False):
        res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, dtype, gate, post, device)
        ro, _, stats = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, scale=0.7,
                                         residual_scale=1.25, eps=EPS)
        out = cpt.residual_norm_backward(dro, dx, ro, y, stats, w_pre, w_post=w_post, gate=g,
                                         scale=0.7, residual_scale=1.25)
        check_backward(out, dro, dx, ro, y, stats, w_pre, w_post, g, 0.7, 1.25)
        again = cpt.residual_norm_backward(dro, dx, ro, y, stats, w_pre, w_post=w_post, gate=g,
                                           scale=0.7, residual_scale=1.25)
        assert all(a is None or torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gate", ["channel", "token"])
def test_fp32_weights(device, dtype, gate):
    cpt = _cpt()
    shape = (2, 33, 776)
    res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, torch.float32, gate, True, device)
    out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, eps=EPS)
    check_forward(out, res, y, w_pre, w_post, g, 1.0, 1.0, EPS)
    grads = cpt.residual_norm_backward(dro, dx, out[0], y, out[2], w_pre, w_post=w_post, gate=g)
    assert all(t.dtype == torch.float32 for t in grads[2:])
    check_backward(grads, dro, dx, out[0], y, out[2], w_pre, w_post, g, 1.0, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts(device, dtype):
    """Only the first norm of a model; only the add; no gradient for the stream."""
    cpt = _cpt()
    shape = (2, 5, 520)
    res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, dtype, "channel", True, device)
    ro, x, stats = cpt.residual_norm(res, None, w_pre, eps=EPS)
    assert ro is res
    r64 = res.double()
    exact = r64 * (r64.square().mean(-1, keepdim=True) + EPS).rsqrt() * w_pre.double()
    _close(x, exact, 64 * E * exact.abs(), "x")
    for up in (dro, None):
        out = cpt.residual_norm_backward(up, dx, res, None, stats, w_pre)
        assert out[1] is None and out[3] is None and out[4] is None
        check_backward(out, up, dx, res, None, stats, w_pre, None, None, 1.0, 1.0)
    ro, x, stats = cpt.residual_norm(res, y, None, w_post=w_post, gate=g, scale=-2.0, eps=EPS)
    assert x is None
    check_forward((ro, x, stats), res, y, None, w_post, g, -2.0, 1.0, EPS)
    out = cpt.residual_norm_backward(dro, None, ro, y, stats, None, w_post=w_post, gate=g,
                                     scale=-2.0)
    check_backward(out, dro, None, ro, y, stats, None, w_post, g, -2.0, 1.0)


def test_views(device):
    """Rows apart (a slice of a longer sequence), elements apart, one row for all."""
    cpt = _cpt()
    base = torch.randn(3, 9, 130, device=device).to(torch.bfloat16)
    y = torch.randn(3, 5, 65, device=device).to(torch.bfloat16)
    w = torch.randn(130, device=device).to(torch.bfloat16)[::2]
    for res in (base[:, 2:7, :65], base[:, 2:7, 65:], base[:, 2:7, ::2],
                base[:1, :1, 3:68].expand(3, 5, 65)):
        out = cpt.residual_norm(res, y, w, eps=EPS)
        check_forward(out, res, y, w, None, None, 1.0, 1.0, EPS)
        grads = cpt.residual_norm_backward(res, y, out[0], res, out[2], w)
        check_backward(grads, res, y, out[0], res, out[2], w, None, None, 1.0, 1.0)


def test_zero_rows_and_large_values(device):
    """A row of zeros has the norm 0 (eps holds the root); large values keep their
    digits; a NaN stays in its row."""
    cpt = _cpt()
    res = torch.zeros(4, 256, device=device).to(torch.bfloat16)
    y = res.clone()
    res[1], y[1] = 1e15, -3e14
    res[2, 7] = float("nan")
    w = torch.ones(256, device=device).to(torch.bfloat16)
    out = cpt.residual_norm(res, y, w, w_post=w, eps=EPS)
    assert (out[1][0] == 0).all() and (out[1][3] == 0).all() and (out[0][0] == 0).all()
    keep = torch.tensor([0, 1, 3], device=device)
    check_forward((out[0][keep], out[1][keep], out[2][:, keep].contiguous()), res[keep], y[keep],
                  w, w, None, 1.0, 1.0, EPS)
    assert out[1][2].isnan().all()


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
def test_rows_of_less_than_a_vector(device, gate):
    """Fewer columns than a vector."""
    cpt = _cpt()
    for shape in ((3, 4, 5), (2, 700, 7), (1, 9, 2)):
        res, y, dro, dx, w_pre, w_post, g = _inputs(shape, torch.bfloat16, torch.float32, gate,
                                                    True, device)
        out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, eps=EPS)
        check_forward(out, res, y, w_pre, w_post, g, 1.0, 1.0, EPS)
        grads = cpt.residual_norm_backward(dro, dx, out[0], y, out[2], w_pre, w_post=w_post, gate=g)
        check_backward(grads, dro, dx, out[0], y, out[2], w_pre, w_post, g, 1.0, 1.0)


def test_graph(device):
    """Captured and replayed, with other work between the replays."""
    cpt = _cpt()
    res, y, dro, dx, w_pre, w_post, g = _inputs((2, 50, 2056), torch.bfloat16, torch.bfloat16,
                                                "channel", True, device)

    def step():
        out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g)
        return out + cpt.residual_norm_backward(dro, dx, out[0], y, out[2], w_pre, w_post=w_post,
                                                gate=g)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        y.copy_(y.roll(1, 1))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(device):
    cpt = _cpt()
    w = torch.ones(64, device=device, requires_grad=True)
    e = torch.zeros(0, 3, 64, device=device)
    ro, x, stats = cpt.residual_norm(e, e, w.detach())
    assert ro.shape == x.shape == (0, 3, 64)
    out = cpt.residual_norm_backward(e, e, ro, e, stats, w.detach())
    assert (out[2] == 0).all() and out[0].shape == (0, 3, 64)


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
def test_function_against_differences(device, gate):
    """The Function's gradients along random directions against difference
    quotients of the 64-bit definition (step 1e-4: truncation ~1e-8)."""
    cpt = _cpt()
    shape = (2, 6, 88)
    res, y, c1, c2, w_pre, w_post, g = _inputs(shape, torch.float32, torch.float32, gate, True,
                                               device)
    leaves = [t.clone().requires_grad_(True) for t in (res, y, w_pre, w_post)]
    if g is not None:
        leaves.append(g.clone().requires_grad_(True))
    ro, x = cpt.ResidualNormFunction.apply(*leaves[:4], leaves[4] if g is not None else None, 0.8,
                                           0.9, EPS)
    ((ro * c1).sum() + (x * c2).sum()).backward()

    def f(ts):
        r, yy, wp, wq = ts[:4]
        u = yy * (yy.square().mean(-1, keepdim=True) + EPS).rsqrt() * wq
        out = 0.9 * r + 0.8 * (u if g is None else ts[4] * u)
        xx = out * (out.square().mean(-1, keepdim=True) + EPS).rsqrt() * wp
        return (out * c1.double()).sum() + (xx * c2.double()).sum()

    at = [t.detach().double() for t in leaves]
    for i, t in enumerate(leaves):
        step = torch.randn(t.shape, device=device, dtype=torch.float64)
        h = 1e-4
        hi = f(at[:i] + [at[i] + h * step] + at[i + 1:])
        lo = f(at[:i] + [at[i] - h * step] + at[i + 1:])
        want, got = (hi - lo) / (2 * h), (t.grad.double() * step).sum()
        size = (t.grad.double() * step).abs().sum()
        assert (got - want).abs() <= 1e-5 * size, (i, float(got), float(want))


def test_module_chain(device):
    """Two modules in a row as a decoder uses them, against autograd of the same
    expressions in 64 bits; unused outputs."""
    cpt = _cpt()
    torch.manual_seed(1)
    a = cpt.ResidualNorm(96, device=device)
    b = cpt.ResidualNorm(96, post=True, gate="channel", gate_init=0.3, scale=0.5, device=device)
    h = torch.randn(4, 96, device=device, requires_grad=True)
    r, x = a(h)
    r, x = b(r, x * 2)
    (r.square().sum() + x.sin().sum()).backward()
    h2 = h.detach().double().requires_grad_(True)

    def rms(t):
        return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()

    r2 = h2 + 0.5 * 0.3 * rms(2 * rms(h2))
    (r2.square().sum() + rms(r2).sin().sum()).backward()
    assert torch.allclose(h.grad.double(), h2.grad, rtol=1e-4, atol=1e-5)
    h.grad = None
    r, x = a(h)
    r.sum().backward()                       # x unused
    assert torch.equal(h.grad, torch.ones_like(h))
    h.grad = None
    r, x = b(h, h)
    x.sum().backward()                       # the stream unused
    assert h.grad.isfinite().all() and b.gate.grad is not None


def test_refusals(device):
    cpt = _cpt()
    r = torch.zeros(2, 3, 64, device=device)
    w = torch.ones(64, device=device)
    for bad in (lambda: cpt.residual_norm(r), lambda: cpt.residual_norm(r, r[:1], w),
                lambda: cpt.residual_norm(r, r.half(), w),
                lambda: cpt.residual_norm(r, r, w[:32]),
                lambda: cpt.residual_norm(r, r, w, gate=torch.ones(3, 64, device=device)),
                lambda: cpt.residual_norm(r, r, w, gate=torch.ones(2, 3, 64, device=device)),
                lambda: cpt.residual_norm(r, r, w, w_post=w.half()),
                lambda: cpt.residual_norm(r.half(), r.half(), w.bfloat16()),
                lambda: cpt.residual_norm(r, None, w, residual_scale=2.0),
                lambda: cpt.residual_norm(r.double(), r.double(), w.double()),
                lambda: cpt.residual_norm(torch.zeros(1, 16392, device=device), None,
                                          torch.ones(16392, device=device))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError):
        cpt.residual_norm(r.cpu(), r, w)


# rows of 16 or 32 threads, several to a wavefront, and the first width beyond them;
# row groups past the last row, blocks of a few rows, sums over several groups
NARROW = [(1, 1, 121), (3, 5, 16), (3, 37, 9), (2, 70, 128), (1, 333, 129), (3, 100, 200),
          (2, 2001, 256), (1, 3000, 257), (1, 20000, 72), (2, 35, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape", NARROW)
def test_narrow_rows(device, dtype, gate, shape):
    cpt = _cpt()
    res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, dtype, gate, True, device, seed=3)
    out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, scale=0.7, residual_scale=1.25,
                            eps=EPS)
    check_forward(out, res, y, w_pre, w_post, g, 0.7, 1.25, EPS)
    ro, _, stats = out
    back = cpt.residual_norm_backward(dro, dx, ro, y, stats, w_pre, w_post=w_post, gate=g,
                                      scale=0.7, residual_scale=1.25)
    check_backward(back, dro, dx, ro, y, stats, w_pre, w_post, g, 0.7, 1.25)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(66000, 1, 8), (65540, 2, 40), (131080, 1, 5)])
def test_many_sequences_with_a_gate_each(device, dtype, shape):
    """More sequences than a grid's second extent."""
    cpt = _cpt()
    res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, dtype, "sequence", True, device)
    out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, eps=EPS)
    check_forward(out, res, y, w_pre, w_post, g, 1.0, 1.0, EPS)
    grads = cpt.residual_norm_backward(dro, dx, out[0], y, out[2], w_pre, w_post=w_post, gate=g)
    check_backward(grads, dro, dx, out[0], y, out[2], w_pre, w_post, g, 1.0, 1.0)


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape,dtype", [((2, 2500, 2048), torch.bfloat16),
                                         ((6, 700, 2048), torch.float16),
                                         ((2, 600, 4097), torch.float32),
                                         ((2, 600, 4097), torch.bfloat16),
                                         ((1, 900, 8200), torch.float16),
                                         ((2, 300, 16384), torch.float32),
                                         ((2, 400, 16383), torch.bfloat16),
                                         ((2, 20000, 5), torch.float32)])
def test_many_rows_a_block(device, shape, dtype, gate):
    """More rows than blocks: each goes over several, in both directions."""
    cpt = _cpt()
    res, y, dro, dx, w_pre, w_post, g = _inputs(shape, dtype, dtype, gate, True, device, seed=5)
    out = cpt.residual_norm(res, y, w_pre, w_post=w_post, gate=g, scale=0.7, residual_scale=1.25,
                            eps=EPS)
    check_forward(out, res, y, w_pre, w_post, g, 0.7, 1.25, EPS)
    ro, _, stats = out
    back = cpt.residual_norm_backward(dro, dx, ro, y, stats, w_pre, w_post=w_post, gate=g,
                                      scale=0.7, residual_scale=1.25)
    check_backward(back, dro, dx, ro, y, stats, w_pre, w_post, g, 0.7, 1.25)
