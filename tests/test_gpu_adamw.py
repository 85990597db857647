"""AdamW over lists of tensors against the formula in 64 bits, and 8-bit moments against
their definition.

Tolerances.  A moment in fp32 is two rounded products (one with a rounded constant) and a
sum: 4 x 2^-24 of its terms.  The update is a root, a division and three products: 12 x
2^-24 of itself; a parameter adds its own rounding u and one of fp32.  8-bit codes are
whole numbers, computed here in the same fp32 operations and from there on exactly:
equal."""

import copy

import pytest
import torch

import compact_amd as cpt

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0 ** -24
HP = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 127, 128, 129, 2048, 8191, 8192, 8193, 20000]


def _mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x243F6A89) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x1E3779B1) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _dither(n, seed, step, i):
    key = _mix(torch.tensor((seed * 0x37E15163 + step * 0x6A09E667 + i * 0x3C6EF373)
                            & 0xFFFFFFFF))
    r = _mix((key + torch.arange(n) * 0x1E3779B9) & 0xFFFFFFFF)
    return (r & 0xFFFF).double() / 65536, (r >> 16).double() / 65536


def _decode(code, scale, ebits):
    """Codes and scale bytes, one a 128 elements, as numbers in 64 bits."""
    c = code.long()
    e, f = c >> 3 & ((1 << ebits) - 1), (c & 7).double()
    y = torch.where(e > 0, (8 + f) * 2.0 ** (e - 1).double(), f)
    s = scale.long().repeat_interleave(128)[:c.numel()]
    y = y * 2.0 ** (s - 134).double()
    y = torch.where(s == 255, float("nan"), y)
    return torch.where(c >= 128, -y, y) if ebits == 4 else y


def _encode(x, u, ebits):
    """The definition, block by block, of fp32 x."""
    codes, scales = [], []
    for b, d in zip(x.double().split(128), u.split(128)):
        top = b.abs().max()
        if not bool(b.isfinite().all()):
            codes.append(torch.zeros(b.numel()))
            scales.append(255)
            continue
        s = -133
        if top > 0:
            s = max(s, int(torch.frexp(top).exponent) - 1 - ((1 << ebits) + 1))
        y = b.abs() * 2.0 ** -s
        unit = 2.0 ** (torch.frexp(y).exponent - 4).clamp(min=0).double()
        q = torch.floor(y / unit + d) * unit
        e = (torch.frexp(q).exponent - 4).clamp(min=0)
        m = q / 2.0 ** e.double()
        code = torch.where(m >= 8, (e + 1) * 8 + m - 8, m).clamp(max=(8 << ebits) - 1)
        if ebits == 5:
            code = torch.where(b > 0, code.clamp(min=1), code)
        else:
            code = code + 128 * (b < 0)
        codes.append(code)
        scales.append(s + 134)
    return torch.cat(codes).to(torch.uint8), torch.tensor(scales, dtype=torch.uint8)


def _make(sizes, dt, gdt, seed=0, gsize=1e-2):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=g).to(dt) for n in sizes]
    grads = [(gsize * torch.randn(n, generator=g) * torch.randn((), generator=g).exp()).to(gdt)
             for n in sizes]
    m = [1e-2 * torch.randn(n, generator=g) for n in sizes]
    v = [1e-4 * torch.rand(n, generator=g) for n in sizes]
    return p, grads, m, v


def _moments(g, m, v, scale=1.0, clip=1.0, hp=HP):
    """m and v of a step in the fp32 operations of its definition."""
    b1, b2 = hp["betas"]
    g = g.float() * scale * clip
    return b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * (g * g)


def _param(p, m, v, t, hp=HP):
    """(p, update) in 64 bits from the moments."""
    b1, b2 = hp["betas"]
    up = hp["lr"] * (m.double() / (1 - b1 ** t)) / ((v.double() / (1 - b2 ** t)).sqrt() + hp["eps"])
    return p.double() * (1 - hp["lr"] * hp["weight_decay"]) - up, up


def _close_param(got, want, up, dt):
    tol = torch.finfo(dt).eps / 2 * want.abs() + 2 * U * want.abs() + 12 * U * up.abs() + 1e-45
    tol += torch.finfo(dt).tiny * torch.finfo(dt).eps
    assert ((got.cpu().double() - want).abs() <= tol).all()


def _to(ts, device):
    return [t.to(device) for t in ts]


@pytest.mark.parametrize("dtype,gtype", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"),
                                         ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("clip", [None, 0.05, 1e6])
def test_float32_moments(device, dtype, gtype, master, clip):
    if master and dtype == "fp32":
        pytest.skip("fp32 parameters have no copy")
    dt, t, scale = TYPES[dtype], 3, 0.5
    sizes = SIZES + [0] + [300] * 50        # over one launch's tensors
    p, g, m, v = _make(sizes, dt, TYPES[gtype])
    copies = [x.float() + 1e-4 for x in p] if master else None
    pd, gd, md, vd = (_to(x, device) for x in (p, g, m, v))
    cd = _to(copies, device) if master else None
    norm = cpt.adamw_step(pd, gd, md, vd, t, masters=cd, grad_scale=scale, max_norm=clip, **HP)
    c = 1.0
    if clip is None:
        assert norm is None
    else:
        want = torch.cat([x.float() * scale for x in g]).double().norm()
        assert abs(float(norm) - want) <= U * want
        c = min(1.0, clip / (float(want) + 1e-6))
    for i in range(len(sizes)):
        m1, v1 = (HP["betas"][0] * m[i].double() + 0.1 * g[i].double() * scale * c,
                  0.95 * v[i].double() + 0.05 * (g[i].double() * scale * c) ** 2)
        size = 0.9 * m[i].double().abs() + 0.1 * g[i].double().abs() * scale * c
        # clip and norm are fp32 too: three roundings more of g, six of g^2
        assert ((md[i].cpu().double() - m1).abs() <= 8 * U * size + 1e-45).all()
        assert ((vd[i].cpu().double() - v1).abs() <= 12 * U * v1 + 1e-45).all()
        if clip is None:        # each operation rounded by itself: the same bits anywhere
            same = _moments(g[i], m[i], v[i], scale)
            assert torch.equal(md[i].cpu(), same[0]) and torch.equal(vd[i].cpu(), same[1])
        want, up = _param(copies[i] if master else p[i], md[i].cpu(), vd[i].cpu(), t)
        _close_param(pd[i], want, up, dt)
        if master:
            _close_param(cd[i], want, up, torch.float32)
            assert torch.equal(pd[i], cd[i].to(dt))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_8bit_moments(device, dtype):
    """Codes, scales and what they stand for, over two steps from zeros."""
    dt = TYPES[dtype]
    p, g, _, _ = _make(SIZES, dt, dt, seed=4)
    g[4][0] = 300.0                          # its block's others are far below
    g[5][128] = 0.0                          # a block of zeros
    pd = _to(p, device)
    code = [[torch.zeros(n, dtype=torch.uint8) for n in SIZES] for _ in "mv"]
    scale = [[torch.zeros(-(-n // 128), dtype=torch.uint8) for n in SIZES] for _ in "mv"]
    cd, sd = [_to(c, device) for c in code], [_to(s, device) for s in scale]
    for t in (1, 2):
        cpt.adamw_step(pd, _to(g, device), *cd, t, m_scales=sd[0], v_scales=sd[1], seed=77, **HP)
        for i, n in enumerate(SIZES):
            m1, v1 = _moments(g[i], _decode(code[0][i], scale[0][i], 4).float(),
                              _decode(code[1][i], scale[1][i], 5).float())
            want, up = _param(p[i], m1, v1, t)
            _close_param(pd[i], want, up, dt)
            p[i] = pd[i].cpu()
            for j, (x, u, e) in enumerate(zip((m1, v1), _dither(n, 77, t, i), (4, 5))):
                code[j][i], scale[j][i] = _encode(x, u, e)
                assert torch.equal(cd[j][i].cpu(), code[j][i]), (t, n, j)
                assert torch.equal(sd[j][i].cpu(), scale[j][i])
            assert (_decode(code[1][i], scale[1][i], 5)[v1 > 0] > 0).all()
        m, v = cpt.adamw_8bit_values(*cd, *sd)
        for i in range(len(SIZES)):
            assert torch.equal(m[i].cpu().double(), _decode(code[0][i], scale[0][i], 4))
            assert torch.equal(v[i].cpu().double(), _decode(code[1][i], scale[1][i], 5))


def test_8bit_rounding_is_fair(device):
    """Over seeds, codes average to the value: at most a step apart, 2^-4 of it, so that
    the mean of 400 lies within 6 x 2^-4 / sqrt(400) / 2 of it; values do not collapse."""
    n = 4096
    g = torch.randn(n, generator=torch.Generator().manual_seed(1)).abs() + 0.5
    total = torch.zeros(n, dtype=torch.float64)
    want = _moments(g, torch.zeros(n), torch.zeros(n))
    sums = [total.clone(), total.clone()]
    for seed in range(400):
        c = [torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(2)]
        s = [torch.zeros(n // 128, dtype=torch.uint8, device=device) for _ in range(2)]
        cpt.adamw_step([torch.zeros(n, device=device)], [g.to(device)], c[:1], c[1:], 1,
                       m_scales=s[:1], v_scales=s[1:], seed=seed, **HP)
        for j in range(2):
            sums[j] += _decode(c[j].cpu(), s[j].cpu(), 4 + j)
    for j in range(2):
        rel = (sums[j] / 400 / want[j].double() - 1)
        # the block's largest may saturate at 15/16 of its binade's end
        low = want[j] < want[j].view(-1, 128).amax(1).repeat_interleave(128) * 0.9
        assert rel[low].abs().max() <= 6 * 0.125 / 2 / 20
        assert rel[low].mean().abs() <= 6 * 0.125 / 2 / 20 / n ** 0.5 + 2.0 ** -16


def test_8bit_extremes(device):
    """Values at both ends of fp32, denormals, blocks that are not finite."""
    n = 128 * 6
    g = torch.randn(n, generator=torch.Generator().manual_seed(2))
    for b, f in enumerate((1e18, 1e-18, 1e-36, 1e-44, 1.0, 1.0)):
        g[b * 128:(b + 1) * 128] *= f
    g[4 * 128 + 3] = float("inf")
    g[5 * 128 + 9] = float("nan")
    p = torch.ones(n)
    c = [torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(2)]
    s = [torch.zeros(6, dtype=torch.uint8, device=device) for _ in range(2)]
    pd = p.to(device)
    cpt.adamw_step([pd], [g.to(device)], c[:1], c[1:], 1, m_scales=s[:1], v_scales=s[1:], seed=5,
                   **HP)
    want = _moments(g, torch.zeros(n), torch.zeros(n))
    for j, (x, u) in enumerate(zip(want, _dither(n, 5, 1, 0))):
        code, scale = _encode(x, u, 4 + j)
        assert torch.equal(s[j].cpu(), scale) and torch.equal(c[j].cpu(), code)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[4 * 128 + 3] = bad[5 * 128 + 9] = True
    assert torch.equal(~pd.cpu().isfinite(), bad)
    m, v = cpt.adamw_8bit_values(c[:1], c[1:], s[:1], s[1:])
    assert m[0][4 * 128:].isnan().all() and v[0][4 * 128:].isnan().all()
    cpt.adamw_step([pd], [torch.ones(n, device=device)], c[:1], c[1:], 2, m_scales=s[:1],
                   v_scales=s[1:], seed=5, **HP)
    assert pd[4 * 128:].isnan().all() and pd[:4 * 128].isfinite().all()


def test_unaligned_codes(device):
    """Codes, scales and parameters that start anywhere in memory."""
    n = 700
    g = torch.Generator().manual_seed(5)
    p, grad = torch.randn(n, generator=g).bfloat16(), torch.randn(n, generator=g).bfloat16()
    runs = []
    for off in (0, 1, 3, 13):
        def at(t):
            whole = torch.zeros(t.numel() + 32, dtype=t.dtype, device=device)
            whole[off:off + t.numel()] = t.to(device)
            return whole[off:off + t.numel()]
        c = [at(torch.zeros(n, dtype=torch.uint8)) for _ in range(2)]
        s = [at(torch.zeros(6, dtype=torch.uint8)) for _ in range(2)]
        x, y = at(p), at(grad)
        for t in (1, 2):
            cpt.adamw_step([x], [y], c[:1], c[1:], t, m_scales=s[:1], v_scales=s[1:], seed=2, **HP)
        m, v = cpt.adamw_8bit_values(c[:1], c[1:], s[:1], s[1:])
        runs.append([x.clone(), *(t.clone() for t in c + s), m[0], v[0]])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_layouts(device):
    """Transposed and sliced parameters, gradients that lie otherwise, unaligned starts."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(40, 33, generator=g)
    grad = torch.randn(33, 40, generator=g)
    flat = torch.randn(1000, generator=g)
    p = [base.to(device).t(), flat.to(device)[3:900]]
    gs = [grad.to(device), torch.randn(897, generator=g).to(device)]
    m = [torch.zeros_like(x) for x in p]
    v = [torch.zeros_like(x) for x in p]
    want = [x.cpu().clone() for x in p]
    cpt.adamw_step(p, gs, m, v, 1, **HP)
    for x, y, w, a, b in zip(p, gs, want, m, v):
        m1, v1 = _moments(y.cpu(), torch.zeros(w.shape), torch.zeros(w.shape))
        ref, up = _param(w, m1, v1, 1)
        _close_param(x, ref, up, torch.float32)
        assert torch.equal(a.cpu(), m1) and torch.equal(b.cpu(), v1)
    # what lies around a sliced parameter is left as it was
    whole = flat.to(device)
    part = whole[5:500]
    cpt.adamw_step([part], [torch.ones_like(part)], [torch.zeros_like(part)],
                   [torch.zeros_like(part)], 1, **HP)
    assert torch.equal(whole[:5].cpu(), flat[:5]) and torch.equal(whole[500:].cpu(), flat[500:])
    assert (whole[5:500].cpu() != flat[5:500]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_grad_norm(device, dtype):
    dt = TYPES[dtype]
    sizes = SIZES + [0] + [33] * 70 + [300001]
    g = _make(sizes, dt, dt, seed=8)[1]
    want = torch.cat([x.double() for x in g]).norm()
    got = cpt.grad_norm(_to(g, device))
    assert abs(float(got) - want) <= U * want
    got = cpt.grad_norm(_to(g, device), grad_scale=0.25)
    assert abs(float(got) - want / 4) <= U * want / 4
    if dtype == "fp32":     # squares beyond fp32
        big = [x.to(device) * 1e25 for x in g]
        assert abs(float(cpt.grad_norm(big)) / (float(want) * 1e25) - 1) <= 4 * U
        big[3][5] = float("inf")
        assert float(cpt.grad_norm(big)) == float("inf")
    assert float(cpt.grad_norm([torch.empty(0, dtype=dt, device=device)])) == 0


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_norm_that_is_not_finite_changes_nothing(device, bits8, bad):
    p, g, m, v = (_to(x, device) for x in _make([300, 9000], torch.bfloat16, torch.bfloat16))
    g[1][17] = bad
    kw = {}
    if bits8:
        m, v = ([torch.randint(0, 100, (n,), dtype=torch.uint8, device=device)
                 for n in (300, 9000)] for _ in range(2))
        kw = dict(m_scales=[torch.full((-(-n // 128),), 120, dtype=torch.uint8, device=device)
                            for n in (300, 9000)])
        kw["v_scales"] = [t.clone() for t in kw["m_scales"]]
    count = torch.tensor([4, 5], device=device)
    before = [t.clone() for t in (*p, *m, *v, count)]
    norm = cpt.adamw_step(p, g, m, v, count, max_norm=1.0, **HP, **kw)
    assert not bool(norm.isfinite())
    assert all(torch.equal(a, b) for a, b in zip((*p, *m, *v, count), before))
    g[1][17] = 0
    cpt.adamw_step(p, g, m, v, count, max_norm=1.0, **HP, **kw)
    assert count.tolist() == [5, 6] and not torch.equal(p[0], before[0])


@pytest.mark.parametrize("bits8", [False, True])
def test_steps_on_the_device_and_lists(device, bits8):
    """Host numbers, a tensor of counts, a count each: the same bits; lr on the device."""
    sizes = [500] * 60
    p, g, m, v = _make(sizes, torch.bfloat16, torch.bfloat16, seed=6)
    t = [1 + i % 7 for i in range(60)]
    runs = []
    for step in (list(t), torch.tensor([x - 1 for x in t], device=device),
                 [torch.tensor(x - 1, device=device) for x in t]):
        args = [_to(x, device) for x in (p, g, m, v)]
        kw = {}
        if bits8:
            args[2:] = ([torch.zeros(500, dtype=torch.uint8, device=device) for _ in sizes]
                        for _ in range(2))
            kw = {n: [torch.zeros(4, dtype=torch.uint8, device=device) for _ in sizes]
                  for n in ("m_scales", "v_scales")}
        lr = HP["lr"] if isinstance(step, list) else torch.tensor(HP["lr"], device=device)
        cpt.adamw_step(*args, step, seed=9, max_norm=0.5, **{**HP, "lr": lr}, **kw)
        runs.append([*args[0], *args[2], *args[3], *(x for n in kw.values() for x in n)])
        if not isinstance(step, list):
            assert step.tolist() == t
        elif isinstance(step[0], torch.Tensor):
            assert [int(x) for x in step] == t
    for other in runs[1:]:
        for i, (a, b) in enumerate(zip(runs[0], other)):
            # 1 / (1 - b^t) of two pow()s: the parameters may differ by a rounding
            assert torch.equal(a, b) or (i < 60 and (a.float() - b.float()).abs().max() <= 0.05)


def _model(dt, device, seed=0):
    torch.manual_seed(seed)
    net = torch.nn.Sequential(torch.nn.Linear(40, 70), torch.nn.LayerNorm(70),
                              torch.nn.Linear(70, 30, bias=False))
    return net.to(device=device, dtype=dt)


def _grads(net, i):
    g = torch.Generator().manual_seed(100 + i)
    for p in net.parameters():
        p.grad = torch.randn(p.shape, generator=g).to(p.device, p.dtype)


def test_optimizer_follows_torchs(device):
    """Ten fp32 steps with two groups: each step's update is good to 24 x 2^-24 and
    parameters to a rounding, ten steps of lr."""
    a, b = _model(torch.float32, device), _model(torch.float32, device)
    groups = [[{"params": list(n[:2].parameters()), "weight_decay": 0.0},
               {"params": list(n[2].parameters()), "lr": 1e-2}] for n in (a, b)]
    opt = cpt.AdamW(groups[0], lr=3e-3, weight_decay=0.1)
    ref = torch.optim.AdamW(groups[1], lr=3e-3, weight_decay=0.1, foreach=False)
    for i in range(10):
        _grads(a, i)
        _grads(b, i)
        if i == 4:      # a parameter without a gradient keeps its own step count
            a[1].bias.grad = b[1].bias.grad = None
        opt.step()
        ref.step()
    for x, y in zip(a.parameters(), b.parameters()):
        assert (x - y).abs().max() <= 10 * (2 * U * y.abs().max() + 24 * U * 1e-2 * 5)


@pytest.mark.parametrize("state", ["float32", "8bit"])
@pytest.mark.parametrize("master", [False, True])
def test_state_dict(device, state, master):
    """A saved and loaded optimizer goes on as the first one, its state in its types."""
    kw = dict(lr=1e-2, state=state, master=master, max_norm=1.0, seed=3)
    a, b = _model(torch.bfloat16, device), _model(torch.bfloat16, device)
    oa, ob = cpt.AdamW(a.parameters(), **kw), cpt.AdamW(b.parameters(), **kw)
    for i in range(3):
        _grads(a, i)
        oa.step()
    b.load_state_dict(a.state_dict())
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))
    for x, y in zip(a.parameters(), b.parameters()):
        sa, sb = oa.state[x], ob.state[y]
        assert sa.keys() == sb.keys() and sb["step"] == 3
        for n in sa:
            if isinstance(sa[n], torch.Tensor):
                assert sa[n].dtype == sb[n].dtype and torch.equal(sa[n], sb[n])
                assert sa[n].data_ptr() != sb[n].data_ptr()
    for i in range(3, 6):
        for net, opt in ((a, oa), (b, ob)):
            _grads(net, i)
            opt.step()
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))
    # the clip is over all tensors, of the step's own gradients
    want = torch.cat([p.grad.double().flatten() for p in a.parameters()]).norm()
    assert abs(float(oa.norm) - float(want)) <= U * float(want)


def test_copies_and_torchs_state(device):
    """A copied optimizer goes on as the first; a state of torch's AdamW is taken."""
    kw = dict(lr=1e-2, max_norm=1.0, seed=3, state="8bit")
    a = _model(torch.bfloat16, device)
    _grads(a, 0)
    opt = cpt.AdamW(a.parameters(), **kw)
    opt.step()
    pair = copy.deepcopy((a, opt))
    for net, o in ((a, opt), pair):
        _grads(net, 1)
        o.step()
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), pair[0].parameters()))
    assert float(pair[1].norm) == float(opt.norm)
    b, c = _model(torch.float32, device), _model(torch.float32, device)
    ref = torch.optim.AdamW(b.parameters(), lr=1e-2, weight_decay=0.1)
    for i in range(2):
        _grads(b, i)
        ref.step()
    for capturable in (False, True):
        c.load_state_dict(b.state_dict())
        own = cpt.AdamW(c.parameters(), lr=1e-2, weight_decay=0.1, capturable=capturable)
        saved = copy.deepcopy(ref.state_dict())
        saved["param_groups"][0]["capturable"] = capturable
        own.load_state_dict(saved)
        _grads(c, 5)
        own.step()
        d = copy.deepcopy(b)
        there = torch.optim.AdamW(d.parameters(), lr=1e-2, weight_decay=0.1, foreach=False)
        there.load_state_dict(copy.deepcopy(ref.state_dict()))
        _grads(d, 5)
        there.step()
        for x, y in zip(c.parameters(), d.parameters()):
            # one step's update of lr x 5 at most, and a rounding of the parameter each
            assert (x - y).abs().max() <= 4 * U * y.abs().max() + 24 * U * 1e-2 * 5


def test_clipping_over_several_kinds(device):
    """One norm over parameters of two types: as each list clipped by that norm."""
    a = _model(torch.bfloat16, device)
    a[1].float()
    b = copy.deepcopy(a)
    _grads(a, 1)
    _grads(b, 1)
    opt = cpt.AdamW(a.parameters(), lr=1e-2, max_norm=0.5)
    opt.step(grad_scale=0.5)
    want = torch.cat([p.grad.double().flatten() for p in b.parameters()]).norm() * 0.5
    assert abs(float(opt.norm) - float(want)) <= 8 * U * float(want)
    for dt in (torch.bfloat16, torch.float32):
        ps = [p for p in b.parameters() if p.dtype == dt]
        z = [[torch.zeros_like(p, dtype=torch.float32) for p in ps] for _ in range(2)]
        with torch.no_grad():
            cpt.adamw_step(ps, [p.grad for p in ps], *z, 1, lr=1e-2, grad_scale=0.5, max_norm=0.5,
                           norm=opt.norm)
    assert all(torch.equal(x, y) for x, y in zip(a.parameters(), b.parameters()))


@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_captured_step(device, state):
    """A graph of a step, replayed with new gradients and another learning rate: as eager."""
    kw = dict(state=state, max_norm=1.0, capturable=True, master=True)
    nets = [_model(torch.bfloat16, device) for _ in range(2)]
    lrs = [torch.tensor(1e-2, device=device) for _ in range(2)]
    opts = [cpt.AdamW(n.parameters(), lr=lr, **kw) for n, lr in zip(nets, lrs)]
    for net, opt in zip(nets, opts):
        _grads(net, 0)
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for i in range(1, 5):
        g = torch.Generator().manual_seed(i)
        for x, y in zip(*(n.parameters() for n in nets)):
            new = torch.randn(x.shape, generator=g).to(x.device, x.dtype)
            x.grad.copy_(new)
            y.grad = new
        for lr in lrs:
            lr.fill_(1e-2 / i)
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        for x, y in zip(*(n.parameters() for n in nets)):
            assert torch.equal(x, y)
            for n, t in opts[0].state[x].items():
                assert torch.equal(t, opts[1].state[y][n]), n
    fresh = cpt.AdamW(_model(torch.float32, device).parameters(), capturable=True)
    host = cpt.AdamW(nets[1].parameters())
    _grads(nets[1], 9)
    host.step()
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            host.step()
    for p in fresh.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()


def test_streams_and_repeated_bits(device):
    p, g, m, v = _make([70000, 12345], torch.bfloat16, torch.bfloat16, seed=5)
    runs = []
    for i in range(3):
        args = [_to(x, device) for x in (p, g, m, v)]
        s = torch.cuda.Stream() if i else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            norm = cpt.adamw_step(*args, 5, max_norm=0.1, **HP)
        torch.cuda.synchronize()
        runs.append([*args[0], *args[2], *args[3], norm])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_elements_past_32_bits(device):
    """The end of a tensor of over 2^32 elements, by its own numbers and the dither of its
    place (of which 32 bits count), and its norm."""
    n, tail = (1 << 32) + 128 * 5 + 77, 128 * 3 + 77
    g = torch.zeros(n, dtype=torch.bfloat16, device=device)
    part = (1e-2 * torch.randn(tail, generator=torch.Generator().manual_seed(3))).bfloat16()
    g[-tail:] = part.to(device)
    p = torch.ones(n, dtype=torch.bfloat16, device=device)
    c = [torch.zeros(n, dtype=torch.uint8, device=device) for _ in range(2)]
    s = [torch.zeros(-(-n // 128), dtype=torch.uint8, device=device) for _ in range(2)]
    norm = cpt.adamw_step([p], [g], c[:1], c[1:], 1, m_scales=s[:1], v_scales=s[1:], seed=4,
                          max_norm=1e6, **HP)
    want = part.double().norm()
    assert abs(float(norm) - want) <= U * want
    m1, v1 = _moments(part, torch.zeros(tail), torch.zeros(tail))
    up = _param(torch.ones(tail), m1, v1, 1)
    _close_param(p[-tail:], *up, torch.bfloat16)
    # elements from 2^32 + 256 on: their low 32 bits
    for j, (x, u) in enumerate(zip((m1, v1), _dither(256 + tail, 4, 1, 0))):
        code, scale = _encode(x, u[256:], 4 + j)
        assert torch.equal(c[j][-tail:].cpu(), code) and torch.equal(s[j][-4:].cpu(), scale)
    assert not c[0][:-tail].any()
