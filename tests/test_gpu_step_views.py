"""Rotation in place and scores over views of one buffer, on the device."""

import pytest
import torch

import compact_amd as cpt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("cut", ["columns", "heads in turn", "tokens in turn", "sequences"])
def test_rotation_in_place_of_heads_side_by_side(device, norm, cut):
    """As out of place, and nothing else of the buffer is touched."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 50, 6, 64, generator=g).bfloat16().to(device)
    views = {"columns": lambda t: (t[..., :32], t[..., 32:]),
             "heads in turn": lambda t: (t[:, :, 0:4:2], t[:, :, 1:4:2]),
             "tokens in turn": lambda t: (t[:, ::2, :5], t[:, 1::2, :5]),
             "sequences": lambda t: (t[:2], t[2:])}[cut]
    q, k = views(x)
    d = q.shape[-1]
    inv = (10000.0 ** (-torch.arange(0, d, 2) / d)).to(device)
    kw = {}
    if norm:
        kw = dict(zip(("w_q", "w_k"), (1 + 0.1 * torch.randn(2, d, generator=g)).to(device)))
    pos = torch.randint(0, 9000, q.shape[:2], generator=g).to(device)
    want = x.clone()
    for t, new in zip(views(want), cpt.qk_rope(q, k, pos, inv, **kw)):
        t.copy_(new)
    assert not torch.equal(want, x)
    cpt.qk_rope(q, k, pos, inv, inplace=True, **kw)
    assert torch.equal(x, want)


def test_a_score_in_place_of_a_computed_view(device):
    """Logits that are a view of a computed tensor give up their memory: the gradient of
    their root is that without inplace; a view of a parameter keeps its own."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 7, 200, generator=g).to(device)
    y = torch.randint(0, 200, (3, 6), generator=g).to(device)
    grads = []
    for inplace in (False, True):
        leaf = x.clone().requires_grad_(True)
        lp, h, *_ = cpt.token_scores((leaf * 1.0)[:, :-1], y, inplace=inplace)
        (lp.sum() - 0.1 * h.sum()).backward()
        assert torch.equal(leaf.detach(), x)
        grads.append(leaf.grad)
    assert torch.equal(*grads) and not grads[0][:, -1].any() and grads[0].any()
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="leaf"):
        cpt.token_scores(leaf[:, :-1], y, inplace=True)
    cpt.token_scores(leaf[:, :-1], y)[0].sum().backward()
    assert torch.equal(leaf.detach(), x)
