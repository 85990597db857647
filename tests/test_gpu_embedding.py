"""The embedding lookup and its gradient against their definitions in 64 bits.

Lookup: one fp32 product, rounded once: the same bits as torch's.
Gradient: |error| <= u |exact| + n_v 2^-24 sum |terms|: u one unit in the output type's
last place, n_v the tokens of a row (an fp32 sum of n_v terms in any order).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}


def _cpt():
    import compact_amd
    return compact_amd


def _ids(kind, n, v, gen):
    if kind == "uniform":
        return torch.randint(0, v, (n,), generator=gen)
    if kind == "one":                      # every token the same
        return torch.full((n,), v // 2)
    if kind == "skewed":                   # a few frequent tokens among rare ones
        r = torch.rand(n, generator=gen)
        return (v * r ** 6).long().clamp(max=v - 1)
    if kind == "outside":
        return torch.randint(-v, 2 * v, (n,), generator=gen)
    raise ValueError(kind)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [torch.int64, torch.int32])
@pytest.mark.parametrize("shape,v,d", [((1,), 1, 1), ((4,), 320, 4096), ((3, 5), 77, 1001),
                                       ((2, 1, 9), 50, 8), ((0,), 5, 16), ((700,), 33, 63)])
def test_lookup(device, dtype, wide, shape, v, d):
    cpt = _cpt()
    g = torch.Generator().manual_seed(d)
    w = torch.randn(v, d, generator=g).to(dtype).to(device)
    n = int(torch.tensor(shape).prod())
    ids = _ids("outside", n, v, g).view(shape).to(wide).to(device)
    for scale in (1.0, d ** 0.5):
        got = cpt.embedding(ids, w, scale)
        ok = ((ids >= 0) & (ids < v)).unsqueeze(-1)
        ref = (w[ids.long().clamp(0, v - 1)].float() * scale).to(dtype)
        assert got.shape == (*shape, d) and got.dtype == dtype
        assert torch.equal(got, torch.where(ok, ref, torch.zeros_like(ref)))


def test_lookup_strided(device):
    cpt = _cpt()
    w = torch.randn(40, 48, device=device)[:, 3:40].to(torch.bfloat16)
    ids = torch.randint(0, 40, (12, 6), device=device)[:, ::2]
    assert torch.equal(cpt.embedding(ids, w), w[ids])


def _check_grad(got, grad, ids, v, scale, padding, base=None):
    d = grad.shape[-1]
    ids, g = ids.reshape(-1).long(), grad.reshape(-1, d).double() * scale
    ok = (ids >= 0) & (ids < v) & (ids != (-1 if padding is None else padding))
    exact = torch.zeros(v, d, dtype=torch.float64, device=g.device)
    terms, count = exact.clone(), torch.zeros(v, dtype=torch.float64, device=g.device)
    exact.index_add_(0, ids[ok], g[ok])
    terms.index_add_(0, ids[ok], g[ok].abs())
    count.index_add_(0, ids[ok], torch.ones_like(ids[ok], dtype=torch.float64))
    if base is not None:
        exact, terms, count = exact + base.double(), terms + base.double().abs(), count + 1
    u = UNIT[got.dtype]
    bound = u * exact.abs() + TINY[got.dtype] + (count + 1).unsqueeze(1) * 2.0 ** -24 * terms
    bad = (got.double() - exact).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off"
    if base is None:
        assert (got[count == 0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "outside"])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 700, 2048), (7, 300, 512), (33, 4, 1001),
                                   (2048, 257, 64), (2049, 70000, 24), (5000, 1000, 520),
                                   (9000, 500, 100)])
def test_gradient(device, dtype, kind, n, v, d):
    cpt = _cpt()
    g = torch.Generator().manual_seed(n + v + d)
    ids = _ids(kind, n, v, g).to(device)
    grad = torch.randn(n, d, generator=g).to(dtype).to(device)
    padding = None if v == 1 else 0
    got = cpt.embedding_backward(grad, ids, v, 3.5, padding_idx=padding)
    assert got.shape == (v, d) and got.dtype == dtype
    _check_grad(got, grad, ids, v, 3.5, padding)
    again = cpt.embedding_backward(grad, ids.int(), v, 3.5, padding_idx=padding)
    assert torch.equal(got, again)         # no order but the tokens'


@pytest.mark.parametrize("n", [16384, 40000, 100352])
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed"])
def test_gradient_long(device, kind, n):
    cpt = _cpt()
    g = torch.Generator().manual_seed(n)
    ids = _ids(kind, n, 32000, g).to(device)
    grad = torch.randn(n, 192, device=device).to(torch.bfloat16)
    got = cpt.embedding_backward(grad, ids, 32000)
    _check_grad(got, grad, ids, 32000, 1.0, None)
    assert torch.equal(got, cpt.embedding_backward(grad, ids, 32000))


@pytest.mark.parametrize("n,v", [(8192, 500), (8193, 500), (12288, 850000), (16385, 32000),
                                 (20000, 31), (20000, 200), (20000, 300000), (32768, 32000),
                                 (32769, 32000), (5000, 4194304), (5000, 4194305), (40000, 200),
                                 (50000, 70000), (114688, 70000), (114689, 70000)])
def test_gradient_sorts(device, n, v):
    """One to three passes of the sort; the lengths at which another one begins."""
    cpt = _cpt()
    g = torch.Generator().manual_seed(n + v)
    ids = _ids("skewed", n, v, g).to(device)
    grad = torch.randn(n, 8 if v > 10 ** 6 else 40, device=device)
    got = cpt.embedding_backward(grad, ids, v, padding_idx=1)
    _check_grad(got, grad, ids, v, 1.0, 1)


@pytest.mark.parametrize("d", [5, 515, 1001])
def test_ragged_rows_added_to_a_buffer(device, d):
    cpt = _cpt()
    g = torch.Generator().manual_seed(d)
    ids = _ids("skewed", 900, 50, g).to(device)
    grad = torch.randn(900, d, generator=g).to(torch.bfloat16).to(device)
    base = torch.randn(50, d, generator=g).to(device)
    out = cpt.embedding_backward(grad, ids, 50, out=base.clone())
    _check_grad(out, grad, ids, 50, 1.0, None, base)


def test_graph(device):
    """Captured and replayed, with other work between the replays."""
    cpt = _cpt()
    w = torch.randn(700, 264, device=device).to(torch.bfloat16)
    for n in (3000, 17000):
        ids = torch.randint(0, 700, (n,), device=device)
        grad = torch.randn(n, 264, device=device).to(torch.bfloat16)
        cpt.embedding_backward(grad, ids, 700)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cpt.embedding(ids, w, 2.0)
            dw = cpt.embedding_backward(grad, ids, 700)
        for i in range(4):
            ids.copy_(ids.roll(7) // (1 + i % 2))
            want = cpt.embedding(ids, w, 2.0), cpt.embedding_backward(grad, ids, 700)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(dw, want[1])


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16),
                                             (torch.bfloat16, torch.float32),
                                             (torch.float16, torch.float32),
                                             (torch.float32, torch.float32)])
@pytest.mark.parametrize("kind", ["one", "skewed"])
def test_gradient_added_to_a_buffer(device, dtype, out_dtype, kind):
    """Rows without tokens keep their bits; the others take one rounding."""
    cpt = _cpt()
    g = torch.Generator().manual_seed(8)
    n, v, d = 700, 90, 264
    ids = _ids(kind, n, v, g).to(device)
    grad = torch.randn(n, d, generator=g).to(dtype).to(device)
    base = torch.randn(v, d, generator=g).to(out_dtype).to(device)
    out = base.clone()
    assert cpt.embedding_backward(grad, ids, v, 0.5, padding_idx=3, out=out) is out
    _check_grad(out, grad, ids, v, 0.5, 3, base)
    used = torch.zeros(v, dtype=torch.bool, device=device)
    used[ids] = True
    used[3] = False
    assert torch.equal(out[~used], base[~used])


def test_gradient_of_views_and_empty_batches(device):
    cpt = _cpt()
    grad = torch.randn(4, 10, 96, device=device).to(torch.bfloat16)
    ids = torch.randint(0, 20, (4, 10), device=device)
    for view, sub in ((grad[:, 2:7], ids[:, 2:7]), (grad[..., :33], ids),
                      (grad[:, :1].expand(4, 10, 96), ids), (grad[..., ::2], ids)):
        _check_grad(cpt.embedding_backward(view, sub, 20), view, sub, 20, 1.0, None)
    none = cpt.embedding_backward(grad[:0], ids[:0], 20)
    assert none.shape == (20, 96) and (none == 0).all()
    assert (cpt.embedding_backward(grad, torch.zeros_like(ids), 20, padding_idx=0) == 0).all()
    assert (cpt.embedding_backward(grad, ids - 1000, 20) == 0).all()


def test_nan_stays_in_its_row(device):
    cpt = _cpt()
    grad = torch.ones(50, 40, device=device)
    ids = torch.arange(50, device=device) % 10
    grad[13] = float("nan")
    got = cpt.embedding_backward(grad, ids, 10)
    assert got[3].isnan().all() and not got[torch.arange(10, device=device) != 3].isnan().any()


def test_module_and_differences(device):
    """ScaledEmbedding's gradient: along a direction, the difference quotient of
    the 64-bit lookup (linear, so exact up to rounding)."""
    cpt = _cpt()
    torch.manual_seed(0)
    m = cpt.ScaledEmbedding(60, 72, padding_idx=5, scale=72 ** 0.5, device=device)
    ids = torch.randint(0, 60, (3, 17), device=device)
    c = torch.randn(3, 17, 72, device=device)
    out = m(ids)
    assert torch.equal(out, torch.nn.functional.embedding(ids, m.weight) * 72 ** 0.5)
    (out * c).sum().backward()
    step = torch.randn(60, 72, device=device).double()
    step[5] = 0
    f = [((m.weight.double() + s * step)[ids] * 72 ** 0.5 * c.double()).sum() for s in (1, -1)]
    want, got = (f[0] - f[1]) / 2, (m.weight.grad.double() * step).sum()
    scale = (m.weight.grad.double() * step).abs().sum()
    assert (got - want).abs() <= 64 * 2.0 ** -24 * scale
    assert (m.weight.grad[5] == 0).all()


def test_another_stream(device):
    cpt = _cpt()
    s = torch.cuda.Stream()
    ids = torch.randint(0, 100, (3000,), device=device)
    grad = torch.randn(3000, 128, device=device)
    want = cpt.embedding_backward(grad, ids, 100)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cpt.embedding_backward(grad, ids, 100)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals(device):
    cpt = _cpt()
    ids = torch.zeros(4, dtype=torch.int64, device=device)
    w = torch.zeros(10, 8, device=device)
    for bad in (lambda: cpt.embedding(ids.short(), w), lambda: cpt.embedding(ids, w.double()),
                lambda: cpt.embedding(ids, w[0]),
                lambda: cpt.embedding_backward(w, ids, 10),
                lambda: cpt.embedding_backward(w[:4], ids, 10, padding_idx=10),
                lambda: cpt.embedding_backward(w[:4], ids, 10, out=w[:9]),
                lambda: cpt.embedding_backward(w[:4].bfloat16(), ids, 10, out=w.half())):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError):
        cpt.embedding(ids.cpu(), w)


@pytest.mark.parametrize("d", [5, 100, 515])
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "outside"])
@pytest.mark.parametrize("n,v", [(9000, 500), (20011, 37), (40000, 3000), (100352, 32000)])
def test_gradient_of_whole_numbers(device, n, v, kind, d):
    """Sums of small whole numbers are exact in fp32 in any order: equal, so that no
    tile of a long run is lost, added twice or put to another id."""
    cpt = _cpt()
    g = torch.Generator().manual_seed(n + d)
    ids = _ids(kind, n, v, g).to(device)
    grad = torch.randint(-8, 9, (n, d), generator=g).to(device)
    ok = (ids >= 0) & (ids < v) & (ids != 1)
    want = torch.zeros(v, d, dtype=torch.float64, device=device)
    want.index_add_(0, ids[ok], grad[ok].double())
    got = cpt.embedding_backward(grad.float(), ids, v, padding_idx=1)
    assert torch.equal(got.double(), want)
    base = torch.randint(-50, 50, (v, d), generator=g).float().to(device)
    got = cpt.embedding_backward(grad.bfloat16(), ids, v, padding_idx=1, out=base.clone())
    assert torch.equal(got.double(), want + base.double())
