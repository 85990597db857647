"""The optimizer's states and options, and views that share memory, on the CPU: tensors
are taken for device ones and every library call is recorded and answered with success."""

import contextlib
import copy
import ctypes
import random
import struct

import pytest
import torch

import compact_amd as cpt
from compact_amd import _lib, optim, rope, scoring


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 1024 if name.endswith("_bytes") else 0
        return call

    def steps(self):
        return [a for n, a in self.calls if n == "cpt_adamw"]


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(_lib, "api", lambda: lib)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for mod in (rope, scoring, optim):
        monkeypatch.setattr(mod, "_stream", lambda t: 0)
        monkeypatch.setattr(mod, "_guard", lambda t: contextlib.nullcontext())
    return lib


def _params(*types):
    ps = [torch.nn.Parameter(torch.full((5,), 1.0 + i, dtype=t)) for i, t in enumerate(types)]
    for p in ps:
        p.grad = torch.ones_like(p)
    return ps


def _torch_state(ps, opt=torch.optim.AdamW, **kw):
    """A state dict of torch's optimizer after one step over parameters like ps."""
    own = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p in own:
        p.grad = torch.ones_like(p)
    ref = opt(own, foreach=False, **kw)
    ref.step()
    return ref.state_dict()


@pytest.mark.parametrize("kw", [{"maximize": True}, {"amsgrad": True},
                                {"opt": torch.optim.Adam, "weight_decay": 0.1}])
def test_states_of_another_formula_are_refused(library, kw):
    """What a step here would not do: maximize, amsgrad, decay within the gradient."""
    ps = _params(torch.float32)
    own = cpt.AdamW(ps, lr=0.5)
    before = copy.deepcopy(own.state_dict())
    with pytest.raises(AssertionError):
        own.load_state_dict(_torch_state(ps, **kw))
    assert own.state_dict() == before
    # without decay Adam is AdamW
    own.load_state_dict(_torch_state(ps, opt=torch.optim.Adam))
    assert own.state[ps[0]]["step"] == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_loaded_state_gets_its_fp32_copy(library, dtype):
    """master=True and a state without the copies: the step makes them of the parameters as
    they then are, and steps them."""
    ps = _params(dtype, dtype)
    own = cpt.AdamW(ps, master=True)
    own.load_state_dict(_torch_state(ps))
    with torch.no_grad():       # the model's weights may be loaded after the optimizer's state
        ps[0].mul_(3)
    own.step()
    (call,) = library.steps()
    assert call[3] == 1
    for p in ps:
        s = own.state[p]
        assert s["step"] == 2 and s["exp_avg"].dtype == torch.float32
        assert s["master"].dtype == torch.float32 and torch.equal(s["master"], p.detach().float())
    kept = [own.state[p]["master"] for p in ps]
    own.step()
    assert all(own.state[p]["master"] is m for p, m in zip(ps, kept))


def test_a_captured_step_needs_the_fp32_copy(library, monkeypatch):
    ps = _params(torch.bfloat16)
    own = cpt.AdamW(ps, master=True, capturable=True)
    own.load_state_dict(_torch_state(ps))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a step is captured"):
        own.step()
    assert "master" not in own.state[ps[0]] and not library.steps()


def test_kinds_of_state_go_by_their_parts(library):
    """A state with a part of the caller's own beside one with as many parts, one of them an
    fp32 copy: two lists, each in its form."""
    ps = _params(torch.bfloat16, torch.bfloat16)
    own = cpt.AdamW([{"params": ps[:1]}])
    own.step()
    own.state[ps[0]]["note"] = "kept"
    own.param_groups[0]["params"].append(ps[1])
    own.state[ps[1]].update(own.state[ps[0]], master=ps[1].detach().float(), step=3)
    for n in ("exp_avg", "exp_avg_sq"):
        own.state[ps[1]][n] = torch.zeros(5)
    del own.state[ps[1]]["note"]
    assert len(own.state[ps[0]]) == len(own.state[ps[1]]) == 4
    for order in (1, -1):
        library.calls.clear()
        own.param_groups[0]["params"] = ps[::order]
        own.step()
        assert [a[3] for a in library.steps()] == [0, 1][::order]
    assert own.state[ps[0]]["note"] == "kept" and own.state[ps[1]]["step"] == 5


def test_loading_keeps_each_groups_own_options(library):
    """torch's state says nothing of `state` and `master`: they stay what the groups, not the
    optimizer's defaults, say; moments that came are float32, and so is the group's state."""
    ps = _params(torch.bfloat16, torch.bfloat16, torch.bfloat16)
    groups = [{"params": ps[:1], "master": True}, {"params": ps[1:2], "state": "8bit"},
              {"params": ps[2:]}]
    saved = _torch_state(ps)
    of = saved["param_groups"][0]
    saved["param_groups"] = [{**of, "params": [i]} for i in range(3)]
    del saved["state"][1]           # of a parameter that was not stepped
    own = cpt.AdamW(groups, state="8bit")
    own.load_state_dict(saved)
    assert [(g["state"], g["master"]) for g in own.param_groups] == \
        [("float32", True), ("8bit", False), ("float32", False)]
    own.step()
    assert [tuple(own.state[p]) for p in ps] == \
        [("step", "exp_avg", "exp_avg_sq", "master"),
         ("step", "exp_avg", "exp_avg_sq", "m_scale", "v_scale"), ("step", "exp_avg", "exp_avg_sq")]
    # its own state says all of it
    again = cpt.AdamW([{"params": [p]} for p in ps])
    again.load_state_dict(own.state_dict())
    assert [(g["state"], g["master"]) for g in again.param_groups] == \
        [(g["state"], g["master"]) for g in own.param_groups]


@pytest.mark.parametrize("size", [1e-30, 1.0, 1e19, 6e37])
def test_norms_of_several_lists_join_in_64_bits(library, size):
    """3 and 4 times any size make 5 times it, to a rounding of each and of the sum: as joined
    by what sums each list's squares."""
    def grad_norm(dt, table, count, scale, out, ws, stream):
        rows = (ctypes.c_int64 * (10 * count)).from_address(table)
        kind, load = ((ctypes.c_float, float), None, (ctypes.c_uint16, None))[dt]
        total = 0.0
        for i in range(count):
            for x in (kind * rows[10 * i + 8]).from_address(rows[10 * i + 1]):
                x = load(x) if load else struct.unpack("f", struct.pack("I", x << 16))[0]
                total += (x * scale) ** 2
        ctypes.c_float.from_address(out).value = total ** 0.5
        return 0

    library.cpt_grad_norm = grad_norm
    ps = _params(torch.float32, torch.bfloat16)
    for p, x in zip(ps, (3 * size, 4 * size)):
        p.grad.zero_()
        p.grad[2] = x
    want = sum(float(p.grad.double().norm()) ** 2 for p in ps) ** 0.5
    own = cpt.AdamW(ps, max_norm=1.0)
    own.step()
    assert own.norm.dtype == torch.float32
    assert abs(float(own.norm) - want) <= 2 * 2.0 ** -24 * want
    assert [a[14] for a in library.steps()] == [1, 1]     # the norm is given to each


def test_an_infinite_max_norm_is_taken(library):
    """As torch's clip_grad_norm_ takes it: the norm is measured, nothing is clipped."""
    ps = _params(torch.float32)
    own = cpt.AdamW(ps, max_norm=float("inf"))
    own.step()
    assert library.steps()[0][13] == float("inf") and own.norm is not None
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(AssertionError):
            cpt.AdamW(ps, max_norm=bad)
        with pytest.raises(AssertionError):
            cpt.adamw_step(ps, [p.grad for p in ps], [torch.zeros(5)], [torch.zeros(5)], 1,
                           max_norm=bad)


@pytest.mark.parametrize("bad", [{"state": "4bit"}, {"state": "8Bit"}, {"lr": -1.0},
                                 {"betas": (0.9, 1.0)}, {"eps": -1e-8}, {"weight_decay": -0.1},
                                 {"maximize": True}, {"amsgrad": True}])
def test_a_groups_options_are_checked(library, bad):
    ps = _params(torch.float32, torch.float32)
    with pytest.raises(AssertionError):
        cpt.AdamW([{"params": ps[:1]}, {"params": ps[1:], **bad}])
    own = cpt.AdamW(ps[:1])
    with pytest.raises(AssertionError):
        own.add_param_group({"params": ps[1:], **bad})
    assert len(own.param_groups) == 1
    own.add_param_group({"params": ps[1:], "state": "8bit", "maximize": False})
    own.step()
    assert [a[2] for a in library.steps()] == [0, 1]
    with pytest.raises(TypeError):
        own.add_param_group(ps)


def test_capturable_may_be_changed(library, monkeypatch):
    """Counts move to the device and back with the group's option, whose steps go on from
    them; while a step is captured they cannot."""
    ps = _params(torch.float32, torch.float32)
    own = cpt.AdamW(ps)
    for _ in range(5):
        own.step()
    own.param_groups[0]["capturable"] = True
    own.step()
    counts = [own.state[p]["step"] for p in ps]
    # the library, which is not there, would add one
    assert all(c.dtype == torch.int64 and int(c) == 5 for c in counts)
    assert counts[0].data_ptr() != counts[1].data_ptr()
    own.step()
    assert all(own.state[p]["step"] is c for p, c in zip(ps, counts))
    own.param_groups[0]["capturable"] = False
    own.step()
    assert [own.state[p]["step"] for p in ps] == [6, 6]
    own.param_groups[0]["capturable"] = True
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    n = len(library.steps())
    with pytest.raises(RuntimeError, match="before a step is captured"):
        own.step()
    own.param_groups[0]["capturable"] = False
    with pytest.raises(RuntimeError, match="capturable=True"):
        own.step()
    assert len(library.steps()) == n and own.state[ps[0]]["step"] == 6


def test_moments_without_both_scales_are_refused(library):
    """Each of the two left out, in the wrapper and in the helper that reads the lists."""
    codes = [torch.zeros(20, dtype=torch.uint8)]
    scales = [torch.zeros(1, dtype=torch.uint8)]
    wide = [torch.zeros(20)]
    for a, b in ((scales, None), (None, scales), (None, None)):
        for m in (codes, wide):
            with pytest.raises(AssertionError):
                cpt.adamw_8bit_values(m, m, a, b)
    out = [[torch.zeros(20, dtype=torch.bfloat16)] for _ in range(2)]
    for a, b in ((scales, None), (None, scales)):
        with pytest.raises(AssertionError):
            _lib.lists().adamw_table(*out, codes, codes, a, b, None, 1, False)
    assert not library.calls
    cpt.adamw_8bit_values(codes, codes, scales, scales)
    assert [n for n, _ in library.calls] == ["cpt_adamw_8bit_values"]


@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_steps_of_any_sequence(library, max_norm):
    """Numbers and counts as a list, a tuple or what gives them one by one; one parameter's
    count as a scalar."""
    def call(step, n=2):
        p, g, m, v = ([torch.ones(5) for _ in range(n)] for _ in range(4))
        cpt.adamw_step(p, g, m, v, step, max_norm=max_norm)
        workspace = library.steps()[-1][17]
        return workspace is not None

    for step in ([3, 4], (3, 4), (i for i in (3, 4)), range(3, 5), 3):
        assert call(step) is (max_norm is not None)
    counts = torch.zeros(2, dtype=torch.int64)
    for step in (counts, list(counts.clone().split(1)), iter(counts.clone().split(1))):
        assert call(step)
    assert call(torch.tensor(0), 1) and call([torch.tensor(0)], 1)
    for bad in ((i for i in (3,)), iter([3, 0]), torch.tensor(0), []):
        with pytest.raises(AssertionError):
            call(bad)


def _cut(buf, *starts, n=40):
    return [buf[a:a + n] for a in starts]


def test_a_steps_tensors_lie_apart(library):
    """Views of one buffer that meet anywhere are refused: of one list, of two, of codes and
    scales, of a gradient and what is written; those side by side in any order are taken."""
    def flat(dt=torch.float32, n=400):
        return torch.zeros(n, dtype=dt)

    def call(p, g, m, v, **kw):
        cpt.adamw_step(p, g, m, v, 1, **kw)

    def two(dt=torch.float32):
        return _cut(flat(dt), 0, 40)

    one = flat()
    x, y = flat(), flat()
    call(_cut(one, 0, 40), _cut(one, 80, 120), _cut(one, 160, 200), _cut(one, 240, 280))
    call(_cut(x, 0, 80), two(), _cut(x, 40, 120), _cut(x, 200, 160))     # in turn, backwards
    call(_cut(x, 40, 0), _cut(x, 80, 120), two(), two())
    m = two()
    call(two(), m, m, two())                      # a gradient that is its moment
    p = two()
    call(p, p, two(), two())
    call([flat(n=0), flat()], [flat(n=0), flat()], [x[5:5], flat()], [x[3:3], x])
    grid = flat(n=1600).view(40, 40)              # columns and rows of one matrix apart
    call([grid[:10].t()], [torch.zeros(40, 10)], [grid[10:20].t()], [grid[20:30].t()])
    codes, scales = torch.zeros(100, dtype=torch.uint8), torch.zeros(8, dtype=torch.uint8)
    call(two(), two(), _cut(codes, 0, 50), _cut(torch.zeros_like(codes), 0, 50),
         m_scales=list(scales[:2].split(1)), v_scales=list(scales[2:4].split(1)))
    call(two(), two(), _cut(codes, 0, 50), _cut(codes.clone(), 0, 50),      # between two codes
         m_scales=[codes[49:50], scales[:1]], v_scales=list(scales[1:3].split(1)))
    half = two(torch.bfloat16)
    call(half, two(torch.bfloat16), two(), two(), masters=_cut(x, 0, 40))
    taken = len(library.steps())
    assert taken == 10
    bad = [lambda: call(_cut(one, 0, 39), two(), two(), two()),
           lambda: call(_cut(one, 39, 0), two(), two(), two()),
           lambda: call(two(), two(), _cut(one, 0, 80), _cut(one, 200, 119)),
           lambda: call(two(), two(), _cut(one, 0, 80), _cut(one, 40, 81)),
           lambda: call(_cut(one, 0, 40), two(), two(), _cut(one, 100, 1)),
           lambda: call([one], [flat()], [flat()], [one]),
           lambda: call([one, one[7:9]], [flat(), flat(n=2)], [flat(), flat(n=2)],
                        [flat(), flat(n=2)]),
           lambda: call(two(), two(), _cut(codes, 0, 50), _cut(codes.clone(), 0, 50),
                        m_scales=list(scales[:2].split(1)), v_scales=list(scales[1:3].split(1))),
           lambda: call(two(), two(), _cut(codes, 0, 50), _cut(codes.clone(), 0, 50),
                        m_scales=[codes[89:90], scales[:1]], v_scales=list(scales[1:3].split(1))),
           lambda: call(half, two(torch.bfloat16), _cut(x, 0, 80), two(), masters=_cut(x, 119, 40)),
           lambda: call(_cut(one, 0, 40), _cut(one, 100, 79), two(), two()),
           lambda: call(_cut(one, 0, 40), _cut(one, 40, 100), two(), two()),
           lambda: call(half, [t[:20].view(torch.bfloat16) for t in m], m, two())]
    for i, f in enumerate(bad):
        with pytest.raises(AssertionError, match="memory"):
            f()
            pytest.fail(f"call {i} was taken")
    assert len(library.steps()) == taken


def test_rotation_in_place_takes_heads_that_lie_apart(library):
    """Heads of one buffer side by side along any axis, and columns in turn."""
    x = torch.zeros(3, 8, 6, 16)
    inv = torch.ones(4)
    pairs = [(x[..., :8], x[..., 8:]), (x[:, :, :4], x[:, :, 4:]), (x[:, :, 4:], x[:, :, :4]),
             (x[:, :, ::2], x[:, :, 1::2]), (x[:, :4], x[:, 4:]), (x[:1], x[1:2]),
             (x[:, ::2], x[:, 1::2]), (x[0], x[1]),
             (x.flatten(1, 2)[:, ::2, None], x.flatten(1, 2)[:, 1::2, None]),
             (x[:, :, 0].unsqueeze(2), x[:, :, 1:]),
             (x[:, :, :2].transpose(1, 2), x[:, :, 2:4].transpose(1, 2)),
             (x[..., :8], x.view(3, 8, 12, 8)[:, :, 1::2]),
             (torch.zeros(1, 8, 4, 16), x[:1, :, :3]), (x[:, :0], x[:, :0])]
    for i, (q, k) in enumerate(pairs):
        cpt.qk_rope(q, k, None, inv, inplace=True)
        assert len(library.calls) == i + 1, i


def test_rotation_in_place_refuses_heads_that_meet(library):
    """Views shifted by a token, a sequence, part of a head or both of two axes."""
    x = torch.zeros(3, 8, 6, 16)
    inv = torch.ones(4)
    flat = x.flatten()
    shifted = [flat[a:a + 2 * 8 * 6 * 16].view(2, 8, 6, 16) for a in (0, 8, 16, 40, 96, 100, 768)]
    pairs = [(x[:, :-1], x[:, 1:]), (x[:, 1:], x[:, :-1]), (x[:-1], x[1:]), (x[1:], x[:-1]),
             (x[..., :10], x[..., 6:]), (x[:, :, :4], x[:, :, 3:]), (x[:, :, 3:], x[:, :, :4]),
             (x[:2, 1:], x[1:, :-1]), (x[:, :-1, 2:], x[:, 1:, :4]), (x, x),
             (x[0, :6], x[0, :6].transpose(0, 1)),
             (x[..., :8], x.view(3, 8, 12, 8)[:, :, ::2]), (x[..., :8], x.view(3, 8, 12, 8)),
             *((shifted[0], s) for s in shifted[1:])]
    for i, (q, k) in enumerate(pairs):
        with pytest.raises(AssertionError, match="one place"):
            cpt.qk_rope(q, k, None, inv, inplace=True)
            pytest.fail(f"pair {i} was taken")
    assert not library.calls


def test_a_score_in_place_spares_leaves_and_their_views(library):
    """The gradient may not be written over a parameter, seen whole or in part."""
    w = torch.zeros(4, 64, requires_grad=True)
    y = torch.zeros(4, dtype=torch.int64)
    for z in (w, w[:, :32], w.view(4, 64), w[:, 8:][:, :9], w.unsqueeze(0)[0], w.t()[:4, :4].t()):
        with pytest.raises(RuntimeError, match="leaf"):
            cpt.token_scores(z, y, inplace=True)
        assert not library.calls
        cpt.token_scores(z, y)
        with torch.no_grad():
            cpt.token_scores(z, y, inplace=True)
        library.calls.clear()
    for z in (w * 1.0, (w * 1.0)[:, :32], w.detach()[:, :32], torch.zeros(4, 64)[:, 1:]):
        cpt.token_scores(z, y, inplace=True)[0]
    assert len(library.calls) == 4


def test_a_modules_frequencies_stay(library):
    """Given to the module or changed in it, they are kept through casts and moves; a module
    made without memory gets them with it."""
    own = torch.rand(8, dtype=torch.float64) / 3
    m = cpt.QKNormRope(24, inv_freq=own, norm=False)
    assert m.rotary == 16 and m.inv_freq.dtype == torch.float32
    assert torch.equal(m.inv_freq, own.float())
    for cast in (lambda t: t.half(), lambda t: t.double(), lambda t: t.to(torch.bfloat16),
                 lambda t: t.to("cpu"), copy.deepcopy, lambda t: t.to_empty(device="cpu")):
        assert torch.equal(cast(m).inv_freq, own.float())
    with torch.no_grad():
        m.inv_freq.mul_(0.25)
    assert torch.equal(m.half().inv_freq, own.float() * 0.25)
    plain = cpt.QKNormRope(16)
    plain.inv_freq = plain.inv_freq / 8
    want = plain.inv_freq.clone()
    assert torch.equal(plain.bfloat16().inv_freq, want) and plain.w_q.dtype == torch.bfloat16
    with torch.device("meta"):
        empty = cpt.QKNormRope(24, inv_freq=torch.rand(8, device="cpu")), cpt.QKNormRope(16)
    assert all(t.inv_freq.is_meta for t in (e.to("meta") for e in empty))
    for e, f in zip(empty, (empty[0]._given, cpt.QKNormRope(16).inv_freq)):
        assert torch.equal(e.to_empty(device="cpu").inv_freq, f)
    # what the rotation is called with
    q, k = torch.zeros(1, 2, 3, 24), torch.zeros(1, 2, 1, 24)
    m(q, k)
    args = library.calls[-1][1]
    assert args[17] == m.inv_freq.data_ptr() and args[23] == 16
    for bad in (dict(inv_freq=torch.ones(2, 4)), dict(inv_freq=torch.ones(13)),
                dict(inv_freq=torch.ones(4), rotary=16), dict(inv_freq=torch.ones(0))):
        with pytest.raises(AssertionError):
            cpt.QKNormRope(24, **bad)


def test_the_fused_forward_takes_plain_attentions_alone():
    """With `rope` an attention's own forward does not run: one that differs, or has hooks,
    is refused before anything is computed."""
    from transformers.models.llama.modeling_llama import LlamaAttention
    from compact_amd import distill_step, e2e

    class Other(LlamaAttention):
        def forward(self, *args, **kw):
            return super().forward(*args, **kw)

    class Same(LlamaAttention):
        pass

    cfg = dict(layers=2, hidden=32, inter=48, heads=2, kv_heads=1, vocab=20, seq=4)
    model = e2e.build_llama(cfg, "cpu")
    ids = torch.zeros(1, 4, dtype=torch.int64)
    a = model.model.layers[1].self_attn

    def call(match, kind=AssertionError):
        with pytest.raises(kind, match=match):
            distill_step.forward(model, ids, rope=True)

    call("HIP device", RuntimeError)            # the embedding's, on the CPU
    a.__class__ = Same
    call("HIP device", RuntimeError)
    a.__class__ = Other
    call("Other has a forward")
    a.__class__ = LlamaAttention
    a.forward = lambda *args, **kw: None
    call("forward of its own")
    del a.forward
    for add in (a.register_forward_hook, a.register_forward_pre_hook,
                a.register_full_backward_hook, a.register_full_backward_pre_hook):
        hook = add(lambda *args: None)
        call("hooks")
        hook.remove()
    call("HIP device", RuntimeError)
    model.model.rotary_emb.rope_type = "dynamic"
    call("go by the length")


def test_views_that_lie_apart_are_told_from_those_that_meet():
    """Random views of one buffer against their elements' places: none that meets is taken,
    and of these none that is apart is refused."""
    rng = random.Random(3)
    buf = torch.zeros(6000)
    where = torch.arange(6000)
    seen = [0, 0]

    def strides(shape):
        order = list(range(len(shape)))
        if rng.random() < 0.4:
            rng.shuffle(order)
        out, step = [0] * len(shape), 1
        for axis in reversed(order):
            out[axis] = step
            step = step * shape[axis] + rng.choice([0, 0, 0, 1, 5, step * shape[axis]])
        return out, step

    for _ in range(3000):
        lead, d = [rng.randint(1, 3) for _ in range(rng.choice([1, 2]))], rng.choice([2, 6, 70])
        shapes = [[*lead, rng.randint(1, 3), d] for _ in range(2)]
        (sq, eq), (sk, ek) = strides(shapes[0]), strides(shapes[1])
        if rng.random() < 0.7:
            sk, ek = sq, eq * 2
        if max(eq, ek) > 4000:
            continue
        at = [rng.randrange(0, rng.choice([10, 400, 1900])) for _ in range(2)]
        q, k = (buf.as_strided(n, s, a) for n, s, a in zip(shapes, (sq, sk), at))
        places = [set(where.as_strided(n, s, a).flatten().tolist())
                  for n, s, a in zip(shapes, (sq, sk), at)]
        if any(len(p) < t.numel() for p, t in zip(places, (q, k))):
            assert not rope._apart(q, k)
            continue
        apart = not places[0] & places[1]
        if not rope._nest(sq, shapes[0]) or not rope._nest(sk, shapes[1]):
            assert not rope._apart(q, k)
            continue
        seen[apart] += 1
        assert rope._apart(q, k) is apart, (q.shape, sq, k.shape, sk, at)
    assert min(seen) > 300


@pytest.mark.parametrize("batch", [1, 4])
def test_one_token_of_a_split_projection_in_place(library, batch):
    """Heads viewed from a projection's columns: an axis of one token has a stride of its own
    in each view, which says nothing."""
    x = torch.zeros(batch, 1, 40 * 128)
    q, k = x[..., :4096].view(batch, 1, 32, 128), x[..., 4096:4608].view(batch, 1, 4, 128)
    assert q.stride() != k.stride()
    cpt.qk_rope(q, k, None, torch.ones(64), inplace=True)
    with pytest.raises(AssertionError, match="one place"):
        cpt.qk_rope(q, x[..., 3968:4480].view(batch, 1, 4, 128), None, torch.ones(64), inplace=True)
    assert len(library.calls) == 1
