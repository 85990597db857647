"""What the wrappers of compact_amd.lm refuse, and what they hand to the library,
on the CPU: tensors are taken for device ones and every library call is recorded
and answered with success.  The C ABI's own refusals, which come before any
launch, are called as they are."""

import pytest
import torch

from compact_amd import _lib, kernels as K, lm


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
    monkeypatch.setattr(lm, "_stream", lambda t: 0)
    return lib


def test_cpu_tensors_are_refused():
    t, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: lm.embedding(i, t), lambda: lm.embedding_backward(t, i, 9),
                 lambda: lm.residual_norm(t, t, torch.ones(8)),
                 lambda: lm.distill_topk(t, t[:, :2], torch.zeros(4, 2, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            call()


def test_gate_kinds():
    shape = (3, 5, 16)
    for gate, want in ((None, (0, 15)), (torch.ones(16), (1, 15)), (torch.ones(1, 1, 16), (1, 15)),
                       (torch.ones(3, 1, 16), (2, 5)), (torch.ones(3, 5, 1), (3, 15))):
        assert lm._gate_kind(gate, shape) == want
    for bad in ((5, 16), (3, 5, 16), (3, 1, 1), (5, 1), (1,), (3, 5), (2, 3, 5, 1), ()):
        with pytest.raises(AssertionError):
            lm._gate_kind(torch.ones(bad), shape)
    assert lm._gate_kind(torch.ones(4, 1), (4, 16)) == (3, 4)
    # one column: a channel's gate is one value for all
    assert lm._gate_kind(torch.ones(1), (4, 1)) == (1, 4)


def test_rows_are_read_as_they_lie(library):
    """Views of whole rows go to the library with their strides; others are copied."""
    base = torch.zeros(4, 9, 40)
    w = torch.ones(16)
    for view, ld in ((base[0, :, :16], 40), (base[:, 0, 3:19], 360), (base[0, :1, :16].expand(6, 16), 0),
                     (base[:, 2:5, :16], 16), (base[0, :, :32:2], 16)):
        library.calls.clear()
        lm.residual_norm(view, None, w)
        name, args = library.calls[-1]
        assert name == "cpt_residual_norm" and args[3] == ld, (args[3], ld)
        if ld != 16:
            assert args[2] == view.data_ptr()


def test_logits_are_read_as_they_lie(library):
    z = torch.zeros(3, 6, 50)
    t, i = torch.zeros(3, 5, 2), torch.zeros(3, 5, 2, dtype=torch.int32)
    lm.distill_topk(z[:, :-1], t, i)
    args = library.calls[-1][1]
    assert args[1] == z.data_ptr() and args[2:7] == (15, 50, 5, 300, 50)
    assert args[-3:-1] == (250, 50)          # the gradient is contiguous
    lm.distill_topk(z[:, 1:], t, i, inplace=True)
    args = library.calls[-1][1]
    assert args[1] == args[-4] == z[:, 1:].data_ptr() and args[-3:-1] == (300, 50)
    lm.distill_topk(z.transpose(1, 2)[:, :5], torch.zeros(3, 5, 2), i)
    assert library.calls[-1][1][2:7] == (15, 6, 15, 0, 6)


def test_nothing_is_launched_for_what_is_refused(library):
    z = torch.zeros(4, 50)
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    w = torch.ones(50)
    for bad in (lambda: lm.distill_topk(z, t, i, alpha=0.5),
                lambda: lm.distill_topk(z, t, i, temperature=-1.0),
                lambda: lm.distill_topk(z, t, i.float()),
                lambda: lm.distill_topk(z, t, i, torch.zeros(3, dtype=torch.int64)),
                lambda: lm.distill_topk(z[:1].expand(4, 50), t, i, inplace=True),
                lambda: lm.residual_norm(z, None, None),
                lambda: lm.residual_norm(z, z, w, gate=torch.ones(3, 50)),
                lambda: lm.residual_norm(z, z, w, eps=-1.0),
                lambda: lm.residual_norm_backward(z, None, z, z, torch.zeros(2, 4), w),
                lambda: lm.residual_norm_backward(z, z, z, z, torch.zeros(2, 3), w),
                lambda: lm.embedding(i.to(torch.uint8), z),
                lambda: lm.embedding_backward(z, i, 9)):
        with pytest.raises(AssertionError):
            bad()
    assert not [c for c in library.calls if not c[0].endswith("_bytes")]


@pytest.fixture(scope="module")
def c_abi():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        from compact_amd import build
        build.build()
    return _lib.lib()


def test_c_refusals(c_abi):
    L, p = c_abi, 4096   # a pointer that is never read
    bad = [
        (L.cpt_embedding, (3, p, 10, 8, p, 1, 4, 1.0, p, None), _lib.ERR_DTYPE),
        (L.cpt_embedding, (2, p, 10, -8, p, 1, 4, 1.0, p, None), _lib.ERR_SHAPE),
        (L.cpt_embedding, (2, None, 10, 8, p, 1, 4, 1.0, p, None), _lib.ERR_SHAPE),
        (L.cpt_embedding_backward, (2, 1, p, 8, p, 1, 4, 10, 8, -1, 1.0, 0, p, p, None),
         _lib.ERR_DTYPE),
        (L.cpt_embedding_backward, (2, 2, p, 8, p, 1, 4, 1 << 31, 8, -1, 1.0, 0, p, p, None),
         _lib.ERR_TOO_LARGE),
        (L.cpt_embedding_backward, (2, 2, p, 8, p, 1, 4, 10, 8, -1, 1.0, 0, p, None, None),
         _lib.ERR_SHAPE),
        (L.cpt_residual_norm, (2, 1, p, 8, p, 8, None, p, None, 0, 4, 4, 8, 1.0, 1.0, 0.0, p, p, p,
                               None), _lib.ERR_DTYPE),
        (L.cpt_residual_norm, (2, 2, p, 8, p, 8, None, p, None, 1, 4, 4, 8, 1.0, 1.0, 0.0, p, p, p,
                               None), _lib.ERR_SHAPE),
        (L.cpt_residual_norm, (2, 2, p, 8, p, 8, None, p, p, 2, 5, 2, 8, 1.0, 1.0, 0.0, p, p, p,
                               None), _lib.ERR_SHAPE),
        (L.cpt_residual_norm, (2, 2, p, 8, p, 8, None, p, None, 0, 4, 4, 16385, 1.0, 1.0, 0.0, p,
                               p, p, None), _lib.ERR_TOO_LARGE),
        (L.cpt_residual_norm, (2, 2, p, 8, None, 8, None, p, None, 0, 4, 4, 8, 1.0, 2.0, 0.0, None,
                               p, p, None), _lib.ERR_SHAPE),
        (L.cpt_distill_topk, (2, p, 4, 50, 4, 0, 50, 3, p, 1, p, 2, None, 1, None, -100, 1.0, 1.0,
                              0, 1.0, None, p, p, p, 0, 50, None), _lib.ERR_DTYPE),
        (L.cpt_distill_topk, (2, p, 4, 50, 4, 0, 50, 0, p, 1, p, 2, None, 1, None, -100, 0.0, 1.0,
                              0, 1.0, None, p, p, p, 0, 50, None), _lib.ERR_SHAPE),
        (L.cpt_distill_topk, (2, p, 4, 50, 4, 0, 50, 0, p, 1, p, 2, None, 1, None, -100, 1.0, 0.5,
                              0, 1.0, None, p, p, p, 0, 50, None), _lib.ERR_SHAPE),
        (L.cpt_distill_topk, (2, p, 4, 50, 4, 0, 50, 0, p, 1, p, 2049, None, 1, None, -100, 1.0,
                              1.0, 0, 1.0, None, p, p, p, 0, 50, None), _lib.ERR_TOO_LARGE),
        (L.cpt_distill_topk, (2, p, 4, 600000, 4, 0, 600000, 0, p, 1, p, 2, None, 1, None, -100,
                              1.0, 1.0, 0, 1.0, None, p, p, p, 0, 50, None), _lib.ERR_TOO_LARGE),
        (L.cpt_scale_rows, (2, None, 4, 50, p, 0, None), _lib.ERR_SHAPE),
    ]
    for fn, args, want in bad:
        assert fn(*args) == want, (fn.__name__, args)
    assert L.cpt_embedding_backward_workspace_bytes(-1, 4, 4) == -1
    assert L.cpt_residual_norm_backward_workspace_bytes(4, 4, 16385, 0) == -1
    assert L.cpt_residual_norm_backward_workspace_bytes(0, 0, 64, 0) == 0


def test_no_work_is_no_launch(c_abi):
    L = c_abi
    assert L.cpt_embedding(2, None, 10, 8, None, 1, 0, 1.0, None, None) == _lib.OK
    assert L.cpt_embedding_backward(2, 2, None, 8, None, 1, 0, 0, 8, -1, 1.0, 0, None, None,
                                    None) == _lib.OK
    assert L.cpt_residual_norm(2, 2, None, 8, None, 8, None, 4096, None, 0, 0, 0, 8, 1.0, 1.0, 0.0,
                               None, 4096, None, None) == _lib.OK
    assert L.cpt_scale_rows(2, None, 0, 50, None, 0, None) == _lib.OK


def test_second_derivatives_are_refused(library):
    """Under create_graph a gradient knows what it came from, and what would need its
    own gradient is an error, not a term left out; first derivatives are as ever."""
    ids = torch.tensor([1, 0, 1])
    table = torch.randn(4, 8, requires_grad=True)
    square = lambda t: (t * t).sum()
    out = lm.EmbeddingFunction.apply(ids, table, 2.0)
    grad, = torch.autograd.grad(square(out), table, create_graph=True)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        square(grad).backward()
    # a gradient that does not depend on the table has none
    grad, = torch.autograd.grad(lm.EmbeddingFunction.apply(ids, table).sum(), table,
                                create_graph=True)
    assert not grad.requires_grad

    w, r, y = (torch.randn(s, requires_grad=True) for s in ((8,), (3, 8), (3, 8)))
    for args in ((r, None, w), (r, y, w), (r, y, w, w, w), (r, y, None, w)):
        ro, x = lm.ResidualNormFunction.apply(*args)
        grads = torch.autograd.grad((ro if x is None else x).sum(), [r, w],
                                    create_graph=True)
        assert grads[1].requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            square(grads[1]).backward()
        ro, x = lm.ResidualNormFunction.apply(*args)
        ((ro if x is None else x).sum()).backward()
        assert library.calls[-1][0] == "cpt_residual_norm_backward"

    z = torch.randn(3, 9, requires_grad=True)
    t, i = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64)
    for dtype in (torch.float32, torch.float16):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(lm.distill_loss(z.to(dtype), t, i), z, create_graph=True)
        lm.distill_loss(z.to(dtype), t, i).backward()


def test_grad_out_lies_with_the_logits(library, monkeypatch):
    z, t, i = torch.zeros(4, 50), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    there = torch.ones(4)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 1 if self is there else 0)
    with pytest.raises(AssertionError, match="tensors on"):
        lm.distill_topk(z, t, i, reduction="none", grad_out=there)
    assert not library.calls
    lm.distill_topk(z, t, i, reduction="none", grad_out=torch.ones(4))


def test_embedding_module_of_a_given_table(library):
    table = torch.arange(12.0).view(4, 3)
    m = lm.ScaledEmbedding.from_pretrained(table, padding_idx=-1, scale=3.0)
    assert m.weight.data_ptr() == table.data_ptr() and not m.weight.requires_grad
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (4, 3, 3, 3.0)
    assert torch.equal(table, torch.arange(12.0).view(4, 3))
    m(torch.tensor([1, 2]))
    assert library.calls[-1][1][1] == table.data_ptr() and library.calls[-1][1][7] == 3.0
    assert lm.ScaledEmbedding.from_pretrained(table, freeze=False).weight.requires_grad
    assert "scale=3.0" in repr(m) and "padding_idx=3" in repr(m)
    with pytest.raises(AssertionError):
        lm.ScaledEmbedding.from_pretrained(table[0])


def test_module_refuses_a_gate_of_nothing(library):
    m, h = lm.ResidualNorm(8), torch.zeros(2, 3, 8)
    with pytest.raises(AssertionError, match="block's output"):
        m(h, gate=torch.ones(2, 3, 1))
    assert not library.calls
    m(h)
    m(h, h, gate=torch.ones(2, 3, 1))
    assert [c[0] for c in library.calls] == ["cpt_residual_norm"] * 2


def test_gradients_of_create_graph_are_ones_own(library):
    """They can be changed in place, as other gradients can."""
    ids, table = torch.tensor([1, 0, 1]), torch.randn(4, 8, requires_grad=True)
    w, r, y = (torch.randn(s, requires_grad=True) for s in ((8,), (3, 8), (3, 8)))
    ro, x = lm.ResidualNormFunction.apply(r, y, w, w)
    out = lm.EmbeddingFunction.apply(ids, table)
    loss = (out * out).sum() + ro.sum() + (x * x).sum()
    for grad in torch.autograd.grad(loss, [table, r, y], create_graph=True):
        grad.mul_(0.5)
        assert grad.requires_grad
