"""The optimizer's states and options, and views that share memory, on the CPU: tensors
are taken for device ones and every library call is recorded and answered with success."""

import contextlib
import copy

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
