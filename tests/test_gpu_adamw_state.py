"""The optimizer over several lists, states and options, on the device.  Tolerances as
test_gpu_adamw.py derives them."""

import pytest
import torch

import compact_amd as cpt
from tests.test_gpu_adamw import HP, U, _close_param, _make, _moments, _param, _to

pytestmark = pytest.mark.gpu


def _two(device, dtypes=(torch.float32, torch.float32), sizes=(300, 5000), seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(n, generator=g).to(device, t))
            for n, t in zip(sizes, dtypes)]


def _draw(ps, i, size=1.0):
    g = torch.Generator().manual_seed(50 + i)
    return [(size * torch.randn(p.shape, generator=g)).to(p.device, p.dtype) for p in ps]


@pytest.mark.parametrize("size", [1e-25, 1e-2, 1e20, 1e30])
def test_the_norm_does_not_go_by_the_groups(device, size):
    """One group and two: the same norm to a rounding of each list's, and a step of the same
    clipped gradients (the clip to 3 roundings, the update to 12 more)."""
    one, two = _two(device), _two(device)
    opts = [cpt.AdamW(one, lr=1e-2, max_norm=1.0),
            cpt.AdamW([{"params": [p]} for p in two], lr=1e-2, max_norm=1.0)]
    before = [p.detach().clone() for p in one]
    for ps, opt in zip((one, two), opts):
        for p, g in zip(ps, _draw(ps, 0, size)):
            p.grad = g
        opt.step()
    want = torch.cat([p.grad.double() for p in one]).norm()
    for opt in opts:
        assert abs(float(opt.norm) - float(want)) <= 3 * U * float(want)
    for a, b, old in zip(one, two, before):
        # every update is at most lr, decay lr x 1e-2 |p|
        assert ((a - b).abs() <= 2 * U * old.abs() + 24 * U * 1e-2).all()
        if size > 1e-20:        # below, eps outweighs the gradient's root
            assert (a != old).all()


def test_captured_step_over_two_lists(device):
    """A graph of a clipped step over two types, replayed with eager work between: as eager."""
    types = (torch.float32, torch.bfloat16)
    nets = [_two(device, types) for _ in range(2)]
    opts = [cpt.AdamW(n, lr=1e-2, max_norm=0.5, capturable=True, state="8bit") for n in nets]
    for net, opt in zip(nets, opts):
        for p, g in zip(net, _draw(net, 0)):
            p.grad = g
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for i in range(1, 5):
        for p, q, g in zip(*nets, _draw(nets[0], i, 10.0 ** (i - 2))):
            p.grad.copy_(g)
            q.grad = g.clone()
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        assert torch.equal(opts[0].norm, opts[1].norm)
        for p, q in zip(*nets):
            assert torch.equal(p, q)
            for n, t in opts[0].state[p].items():
                assert torch.equal(t, opts[1].state[q][n]), n


@pytest.mark.parametrize("lists", [1, 2])
def test_an_infinite_max_norm_measures(device, lists):
    """The norm, and the bits of a step without clipping; one that is not finite still
    leaves the step out."""
    a, b = _two(device), _two(device)
    groups = [{"params": [p]} for p in a] if lists == 2 else a
    opt, ref = cpt.AdamW(groups, max_norm=float("inf")), cpt.AdamW(b)
    for i in range(2):
        for x, y, g in zip(a, b, _draw(a, i, 7.0)):
            x.grad, y.grad = g, g.clone()
        opt.step()
        ref.step()
    want = torch.cat([p.grad.double() for p in a]).norm()
    assert abs(float(opt.norm) - float(want)) <= 3 * U * float(want)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    a[0].grad[3] = float("inf")
    opt.step()
    assert float(opt.norm) == float("inf") and all(torch.equal(x, y) for x, y in zip(a, b))


def test_capturable_may_be_changed(device):
    """Steps with host counts, then captured ones, then host counts again: as with host
    counts throughout (1 / (1 - b^t) of two pow()s: the update to 4 roundings)."""
    a, b = _two(device), _two(device)
    opt, ref = cpt.AdamW(a, lr=1e-2), cpt.AdamW(b, lr=1e-2)

    def grads(i):
        for x, y, g in zip(a, b, _draw(a, i)):
            if x.grad is None:
                x.grad = g.clone()
            x.grad.copy_(g)
            y.grad = g

    for i in range(2):
        grads(i)
        opt.step()
        ref.step()
    opt.param_groups[0]["capturable"] = True
    grads(2)
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(3, 6):
        grads(i)
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
    opt.param_groups[0]["capturable"] = False
    grads(6)
    opt.step()
    ref.step()
    for x, y in zip(a, b):
        s, t = opt.state[x], ref.state[y]
        assert s["step"] == t["step"] == 7
        assert torch.equal(s["exp_avg"], t["exp_avg"])
        assert torch.equal(s["exp_avg_sq"], t["exp_avg_sq"])
        # seven updates of 5 lr at most, a rounding of the parameter each
        assert ((x - y).abs() <= 7 * (2 * U * y.abs() + 4 * U * 5e-2)).all()


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("on", ["numbers", "counts", "a count each"])
def test_each_way_of_counting_makes_the_formulas_parameters(device, bits8, on):
    """Clipped bf16 steps at counts of their own: parameters against the formula in 64 bits at
    each tensor's step number and the lr given, from moments computed in the same fp32
    operations."""
    sizes = [500] * 60
    p, g, m, v = _make(sizes, torch.bfloat16, torch.bfloat16, seed=6)
    t = [1 + i % 7 for i in range(60)]
    step = {"numbers": t, "counts": torch.tensor([x - 1 for x in t], device=device),
            "a count each": [torch.tensor(x - 1, device=device) for x in t]}[on]
    kw = {}
    if bits8:
        # codes and scales of any moments do: those that a step leaves
        m, v = ([torch.zeros(500, dtype=torch.uint8) for _ in sizes] for _ in range(2))
        scales = [[torch.zeros(4, dtype=torch.uint8, device=device) for _ in sizes]
                  for _ in range(2)]
        kw = dict(m_scales=scales[0], v_scales=scales[1], seed=9)
    pd, gd, md, vd = (_to(x, device) for x in (p, g, m, v))
    if bits8:
        other = _to(_make(sizes, torch.bfloat16, torch.bfloat16, seed=7)[1], device)
        cpt.adamw_step([x.clone() for x in pd], other, md, vd, 1, **HP, **kw)
        m, v = ([x.cpu().float() for x in y] for y in cpt.adamw_8bit_values(md, vd, *scales))
    hp = {**HP, "lr": 7e-3}
    lr = hp["lr"] if on == "numbers" else torch.tensor(hp["lr"], device=device)
    norm = cpt.adamw_step(pd, gd, md, vd, step, max_norm=0.5, **{**hp, "lr": lr}, **kw)
    clip = (torch.tensor(0.5) / (norm.cpu() + 1e-6)).clamp(max=1.0)
    assert clip < 1
    for i in range(60):
        m1, v1 = _moments(g[i], m[i], v[i], clip=clip)
        if not bits8:
            assert torch.equal(md[i].cpu(), m1) and torch.equal(vd[i].cpu(), v1)
        want, up = _param(p[i], m1, v1, t[i], hp)
        _close_param(pd[i], want, up, torch.bfloat16)


@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_captured_steps_are_the_hosts(device, state):
    """A captured step with counts and lr on the device, replayed with other gradients and
    another lr, against eager steps with numbers: moments and codes the same bits, parameters
    apart by 1 / (1 - b^t) of two pow()s (4 roundings of the update) and their own rounding."""
    a, b = _two(device), _two(device)
    lr = torch.tensor(1e-2, device=device)
    kw = dict(state=state, max_norm=2.0)
    opt, ref = cpt.AdamW(a, lr=lr, capturable=True, **kw), cpt.AdamW(b, lr=1e-2, **kw)

    def step(i, run):
        for x, y, g in zip(a, b, _draw(a, i)):
            x.grad = g.clone() if x.grad is None else x.grad.copy_(g)
            y.grad = g
        ref.param_groups[0]["lr"] = 1e-2 / (1 + i)
        lr.fill_(1e-2 / (1 + i))
        run()
        ref.step()
        torch.cuda.synchronize()

    step(0, opt.step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(1, 6):
        before = [p.detach().clone() for p in b]
        step(i, graph.replay)
        assert torch.equal(opt.norm, ref.norm)
        for x, y, old in zip(a, b, before):
            s, t = opt.state[x], ref.state[y]
            assert int(s["step"]) == t["step"] == i + 1
            assert all(torch.equal(s[n], t[n]) for n in s if n != "step")
            assert ((x - y).abs() <= (i + 1) * (2 * U * y.abs() + 4 * U * 5e-2)).all()
            # the updates are hundreds of these bounds
            assert (y - old).abs().mean() > 1e-4
