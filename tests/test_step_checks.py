"""What the wrappers of rope.py, scoring.py and optim.py refuse, and what they hand to the
library, on the CPU: tensors are taken for device ones and every library call is
recorded and answered with success.  The C ABI's own refusals, which come before any
launch, are called as they are."""

import contextlib
import ctypes

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


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(_lib, "api", lambda: lib)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    for mod in (rope, scoring, optim):
        monkeypatch.setattr(mod, "_stream", lambda t: 0)
        monkeypatch.setattr(mod, "_guard", lambda t: contextlib.nullcontext())
    return lib


def _launches(library):
    return [c for c in library.calls if not c[0].endswith("_bytes")]


def test_cpu_tensors_are_refused():
    q, inv = torch.zeros(1, 2, 3, 8), torch.ones(4)
    z, y = torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64)
    p = [torch.zeros(4)]
    for call in (lambda: cpt.qk_rope(q, q, None, inv),
                 lambda: cpt.qk_rope_backward(q, q, q, q, None, inv, w_q=inv, w_k=inv),
                 lambda: cpt.token_logprobs(z, y), lambda: cpt.grad_norm(p),
                 lambda: cpt.token_logprobs_backward(z, y, z[:, 0], None, z[:, 0]),
                 lambda: cpt.adamw_step(p, p, p, p, 1),
                 lambda: cpt.adamw_8bit_values([t.byte() for t in p], *[[t.byte() for t in p]] * 3)):
        with pytest.raises(RuntimeError):
            call()


def test_optimizer_refuses_cpu_parameters():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    for kw in ({}, {"capturable": True}, {"state": "8bit", "max_norm": 1.0}):
        opt = cpt.AdamW([p], **kw)
        with pytest.raises(RuntimeError, match="HIP device only"):
            opt.step()
        assert not opt.state[p] and torch.equal(p.detach(), torch.zeros(4))


def test_rope_refusals(library):
    q, k, inv = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.ones(8)
    w, pos = torch.ones(16), torch.zeros(2, 5, dtype=torch.int64)
    bad = [lambda: cpt.qk_rope(q, k.half(), pos, inv), lambda: cpt.qk_rope(q, k[:1], pos, inv),
           lambda: cpt.qk_rope(q, k[..., :14], pos, inv), lambda: cpt.qk_rope(q[0, 0], k[0, 0], pos, inv),
           lambda: cpt.qk_rope(q[..., :15], k[..., :15], pos, inv),
           lambda: cpt.qk_rope(q, k, pos.float(), inv), lambda: cpt.qk_rope(q, k, pos[:, :4], inv),
           lambda: cpt.qk_rope(q, k, pos[:, 0], inv), lambda: cpt.qk_rope(q, k, pos, inv.double()),
           lambda: cpt.qk_rope(q, k, pos, torch.ones(9)), lambda: cpt.qk_rope(q, k, pos, torch.ones(0)),
           lambda: cpt.qk_rope(q, k, pos, inv, w_q=w), lambda: cpt.qk_rope(q, k, pos, inv, w_q=w, w_k=w[:8]),
           lambda: cpt.qk_rope(q, k, pos, inv, w_q=w.half(), w_k=w.half()),
           lambda: cpt.qk_rope(q, k, pos, inv, w_q=w, w_k=w, eps=-1.0),
           lambda: cpt.qk_rope(q, k, pos, inv, w_q=w, w_k=w, inverse=True),
           lambda: cpt.qk_rope(q.double(), k.double(), pos, inv),
           lambda: cpt.qk_rope(q[:, :, :0], k, pos, inv),
           lambda: cpt.qk_rope(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos, inv, inplace=True),
           lambda: cpt.qk_rope(q[:, :, :1].expand(2, 5, 4, 16), k, pos, inv, inplace=True),
           lambda: cpt.qk_rope(q, q, pos, inv, inplace=True),
           lambda: cpt.qk_rope(q[:, :, :3], q[:, :, 2:], pos, inv, inplace=True),
           lambda: cpt.qk_rope(q, k, pos[None], inv), lambda: cpt.qk_rope(q[0], k[0], pos[:1], inv),
           lambda: cpt.qk_rope_backward(q, k[:, :, :1], q, k, pos, inv, w_q=w, w_k=w),
           lambda: cpt.qk_rope_backward(q.half(), k, q, k, pos, inv, w_q=w, w_k=w),
           lambda: cpt.QKNormRope(16, rotary=18), lambda: cpt.QKNormRope(16, rotary=7)]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")
    assert not _launches(library)


def test_rope_reads_heads_as_they_lie(library):
    qkv = torch.zeros(3, 7, 8, 32)
    inv = torch.ones(16)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    cpt.qk_rope(q, k, None, inv)
    a = library.calls[-1][1]
    assert a[4:8] == (q.data_ptr(), 1792, 256, 32) and a[8:12] == (k.data_ptr(), 1792, 256, 32)
    assert a[14:17] == (None, 0, 0) and a[18:24] == (3, 7, 4, 2, 32, 32)
    assert a[27:30] == (896, 128, 32) and a[31:34] == (448, 64, 32)
    cpt.qk_rope(q, k, torch.zeros(3, 7, dtype=torch.int32), inv, inplace=True)
    a = library.calls[-1][1]
    assert a[15:17] == (0, 7) and a[26] == q.data_ptr() and a[27:30] == (1792, 256, 32)
    cpt.qk_rope(q[0], k[0], torch.zeros(7, dtype=torch.int64), inv)
    a = library.calls[-1][1]
    assert a[5:8] == (0, 256, 32) and a[15:17] == (1, 0) and a[18:20] == (1, 7)
    cpt.qk_rope(q.transpose(1, 2).contiguous().transpose(1, 2), k, None, inv)
    assert library.calls[-1][1][5:8] == (896, 32, 224)


def test_scoring_refusals(library):
    z, y = torch.zeros(4, 50), torch.zeros(4, dtype=torch.int64)
    f = torch.zeros(4)
    s = torch.zeros(2, 4)
    b = cpt.token_logprobs_backward
    bad = [lambda: cpt.token_logprobs(z, y[:3]), lambda: cpt.token_logprobs(z, y.float()),
           lambda: cpt.token_logprobs(z, y, temperature=0.0),
           lambda: cpt.token_logprobs(z, y, temperature=float("inf")),
           lambda: cpt.token_logprobs(z, y, temperature=float("nan")),
           lambda: cpt.token_logprobs(z, y, top_k=51), lambda: cpt.token_logprobs(z, y, top_k=-1),
           lambda: cpt.token_logprobs(torch.zeros(4, 500), y, top_k=129),
           lambda: cpt.token_logprobs(z.double(), y), lambda: cpt.token_logprobs(z[:, :0], y),
           lambda: cpt.token_logprobs(torch.zeros(()), None),
           lambda: b(z, None, f, f, f), lambda: b(z, y, f, None, f, f), lambda: b(z, y, None, f, f),
           lambda: b(z, y, f[:3], f, f), lambda: b(z, y, f, f, f.half()),
           lambda: b(z, y, f, f, f, stats=s[:, :3]), lambda: b(z, y, f, f, f, stats=s.double()),
           lambda: b(z[:1].expand(4, 50), y, f, f, f, inplace=True),
           lambda: b(torch.zeros(50, 4).t(), y, f, f, f, inplace=True)]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")
    assert not _launches(library)


def test_scoring_reads_logits_as_they_lie(library):
    z, y = torch.zeros(3, 6, 50), torch.zeros(3, 5, dtype=torch.int32)
    cpt.token_logprobs(z[:, :-1], y, top_k=3)
    a = library.calls[-1][1]
    assert a[1:7] == (z.data_ptr(), 15, 50, 5, 300, 50) and a[7] == 0 and a[11] == 3
    f = torch.zeros(3, 5)
    cpt.token_logprobs_backward(z[:, 1:], y, f, f, f, inplace=True)
    a = library.calls[-1][1]
    assert a[1] == a[16] == z[:, 1:].data_ptr() and a[17:19] == (300, 50)


def _adamw_args():
    p = [torch.zeros(5, 4), torch.zeros(300)]
    return p, [torch.ones_like(t) for t in p], [torch.zeros_like(t) for t in p], \
        [torch.zeros_like(t) for t in p]


def test_adamw_refusals(library):
    p, g, m, v = _adamw_args()
    s = cpt.adamw_step
    half = [t.half() for t in p]
    codes = [torch.zeros(20, dtype=torch.uint8), torch.zeros(300, dtype=torch.uint8)]
    scales = [torch.zeros(1, dtype=torch.uint8), torch.zeros(3, dtype=torch.uint8)]
    one = torch.ones(1)
    bad = [lambda: s(p, g[:1], m, v, 1), lambda: s(p, g, m[:1], v, 1), lambda: s(p, g, m, v, 0),
           lambda: s(p, g, m, v, [1]), lambda: s(p, g, m, v, [1, 0]), lambda: s(p, g, m, v, [1, 2.0]),
           lambda: s(p, g, m, v, torch.zeros(3, dtype=torch.int64)),
           lambda: s(p, g, m, v, torch.zeros(2)),
           lambda: s(p, g, m, v, [torch.zeros(1, dtype=torch.int64)] * 2),
           lambda: s(p, g, m, v, 1, lr=-1.0), lambda: s(p, g, m, v, 1, lr=torch.ones(2)),
           lambda: s(p, g, m, v, 1, betas=(1.0, 0.9)), lambda: s(p, g, m, v, 1, betas=(0.9, -0.1)),
           lambda: s(p, g, m, v, 1, eps=-1.0), lambda: s(p, g, m, v, 1, weight_decay=-1.0),
           lambda: s(p, g, m, v, 1, max_norm=0.0), lambda: s(p, g, m, v, 1, norm=one),
           lambda: s(p, g, m, v, 1, max_norm=1.0, norm=one.double()),
           lambda: s(p, g, m, v, 1, m_scales=scales), lambda: s(p, g, m, v, 1, masters=m),
           lambda: s(p, [t.half() for t in g], m, v, 1), lambda: s(p, [g[0], g[1].half()], m, v, 1),
           lambda: s([p[0], half[1]], g, m, v, 1), lambda: s([t.double() for t in p], g, m, v, 1),
           lambda: s(p, [g[0].t(), g[1]], m, v, 1), lambda: s(p, g, half, v, 1),
           lambda: s(p, g, [m[0].t().contiguous().t(), m[1]], v, 1),
           lambda: s([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], 1),
           lambda: s([p[1][::2], p[0]], [g[1][::2], g[0]], [m[1][::2], m[0]], [v[1][::2], v[0]], 1),
           lambda: s(p, g, m, m, 1), lambda: s(p, g, p, v, 1), lambda: s(p, g, m, [v[0], m[1]], 1),
           lambda: s(p, g, codes, codes, 1, m_scales=scales, v_scales=scales[:1]),
           lambda: s(p, g, codes, codes, 1, m_scales=scales, v_scales=scales[::-1]),
           lambda: s(p, g, m, codes, 1, m_scales=scales, v_scales=scales),
           lambda: cpt.grad_norm([]), lambda: cpt.grad_norm([t.double() for t in g]),
           lambda: cpt.grad_norm(g, out=torch.zeros(2)),
           lambda: cpt.adamw_8bit_values(codes, codes[:1], scales, scales),
           lambda: cpt.adamw_8bit_values(m, codes, scales, scales),
           lambda: cpt.AdamW(p, state="4bit"), lambda: cpt.AdamW(p, lr=-1.0),
           lambda: cpt.AdamW(p, betas=(0.9, 1.0)), lambda: cpt.AdamW(p, max_norm=0.0)]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            pytest.fail(f"call {i} was taken")
    assert not _launches(library)
    assert s([], [], [], [], 1) is None


def test_adamw_table(library):
    """Each tensor's addresses, size and step as the C ABI reads them."""
    p, g, m, v = _adamw_args()
    seen = []
    library.cpt_adamw = lambda *a: seen.append(
        (a, list((ctypes.c_int64 * 20).from_address(a[4])))) or 0
    cpt.adamw_step(p, g, m, v, [3, 9], seed=-1)
    a, rows = seen[0]
    assert a[:4] == (0, 0, 0, 0) and a[5] == 2 and a[15] == 0xFFFFFFFF
    for i, t in enumerate((3, 9)):
        assert rows[10 * i:10 * i + 10] == [x[i].data_ptr() for x in (p, g, m, v)] + \
            [0, 0, 0, 0, p[i].numel(), t]
    versions = [t._version for t in p]
    cpt.adamw_step(p, g, m, v, torch.zeros(2, dtype=torch.int64))
    a, rows = seen[1]
    assert rows[17] == rows[7] + 8 and rows[9] == rows[19] == 0
    assert [t._version for t in p] > versions


@pytest.fixture(scope="module")
def c_abi():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from compact_amd import build
        build.build()
    return _lib.lib()


def test_c_refusals(c_abi):
    L, p = c_abi, 4096      # a pointer that is never read
    st = (8, 8, 8)
    pos = (None, 0, 0, p)

    def rope_call(dt=2, wdt=2, inverse=0, w=(None, None), b=1, s=1, d=8, r=8, eps=1e-6, q=p):
        return L.cpt_qk_rope(dt, wdt, 0, inverse, q, *st, p, *st, *w, *pos, b, s, 2, 2, d, r, eps,
                             1.0, p, *st, p, *st, None)

    assert rope_call(dt=3) == _lib.ERR_DTYPE and rope_call(wdt=1) == _lib.ERR_DTYPE
    assert rope_call(d=7) == rope_call(r=10) == rope_call(r=3) == rope_call(b=-1) == _lib.ERR_SHAPE
    assert rope_call(w=(p, None)) == rope_call(inverse=1, w=(p, p)) == _lib.ERR_SHAPE
    assert rope_call(eps=-1.0) == rope_call(eps=float("nan")) == rope_call(q=None) == _lib.ERR_SHAPE
    assert rope_call(d=1026, r=8) == rope_call(b=1 << 20, s=1 << 20) == _lib.ERR_TOO_LARGE
    assert rope_call(s=0) == _lib.OK
    args = (2, 2, 0, p, *st, p, *st, p, *st, p, *st)
    tail = (1, 1, 2, 2, 8, 8, 1e-6, 1.0)
    assert L.cpt_qk_rope_backward(*args, None, p, *pos, *tail, p, p, p, p, p, None) == _lib.ERR_SHAPE
    assert L.cpt_qk_rope_backward(*args, p, p, *pos, *tail, p, p, p, p, None, None) == _lib.ERR_SHAPE
    assert L.cpt_qk_rope_backward_workspace_bytes(4, 2, 2, 2000) == -1

    def lp(dt=2, rows=4, v=50, t=1.0, k=2, y=p, lpp=p, top=p):
        return L.cpt_token_logprobs(dt, p, rows, v, 4, 0, v, 1, y, -100, t, k, lpp, p, p, p, top,
                                    top, None)

    assert lp(dt=5) == _lib.ERR_DTYPE
    assert lp(t=1e-39) == lp(v=0) == lp(t=0.0) == lp(t=float("inf")) == lp(k=51) == lp(y=None) == _lib.ERR_SHAPE
    assert lp(top=None) == lp(rows=-1) == _lib.ERR_SHAPE
    assert lp(v=500, k=129) == lp(v=1 << 25) == lp(rows=1 << 31) == _lib.ERR_TOO_LARGE
    assert lp(rows=0) == _lib.OK

    def lg(dt=2, y=p, lse=p, h=p, a=p, b=p):
        return L.cpt_token_logprobs_backward(dt, p, 4, 50, 4, 0, 50, 1, y, -100, 1.0, lse, None, h,
                                             a, b, None, 0, 50, None)

    assert lg(dt=-1) == _lib.ERR_DTYPE and lg() == lg(lse=None) == lg(h=None) == _lib.ERR_SHAPE

    def table(**kw):
        f = dict(zip(("p", "g", "m", "v", "ms", "vs", "master", "sd", "n", "step"),
                     (p, p, p, p, p, p, p, 0, 100, 1)))
        f.update(kw)
        t = (ctypes.c_int64 * 10)(*f.values())
        keep.append(t)
        return ctypes.addressof(t)

    keep = []

    def step(dt=2, gdt=2, bits=0, master=0, t=None, n=1, b1=0.9, eps=1e-8, norm=0.0, ws=p):
        return L.cpt_adamw(dt, gdt, bits, master, t if t is not None else table(), n, 1e-3, None, b1,
                           0.99, eps, 0.0, 1.0, norm, 0, 0, p, ws, None)

    assert step(dt=4) == step(gdt=1) == step(dt=0, gdt=0, master=1) == _lib.ERR_DTYPE
    for f in "pgmv":
        assert step(t=table(**{f: 0})) == _lib.ERR_SHAPE
    assert step(t=table(n=-1)) == step(t=table(step=0)) == step(b1=1.0) == _lib.ERR_SHAPE
    assert step(bits=1, t=table(ms=0)) == step(master=1, t=table(master=0)) == _lib.ERR_SHAPE
    assert step(norm=1.0, ws=None) == step(t=table(sd=p), ws=None) == step(n=-1) == _lib.ERR_SHAPE
    assert step(t=table(n=1 << 41)) == _lib.ERR_TOO_LARGE
    assert step(n=0) == _lib.OK
    assert L.cpt_grad_norm(7, table(), 1, 1.0, p, p, None) == _lib.ERR_DTYPE
    assert L.cpt_grad_norm(2, table(g=0), 1, 1.0, p, p, None) == _lib.ERR_SHAPE
    assert L.cpt_adamw_8bit_values(table(vs=0), 1, None) == _lib.ERR_SHAPE
    assert L.cpt_adamw_8bit_values(None, 0, None) == _lib.OK
    assert L.cpt_adamw_workspace_bytes(-1, 5) == -1 and L.cpt_adamw_workspace_bytes(3, 5) > 0
