"""The rotation, scoring and optimizer as the distillation step uses them together, on a
small LLaMA in float32 (attention and GEMMs are the same calls, so that the two sides
differ by fp32 rounding alone: 1e-4 of a tensor's norm), and bf16 steps with FlashFFN v3
in every MLP and 8-bit moments."""

import pytest
import torch

import compact_amd as cpt
from compact_amd import distill_step as D
from compact_amd import e2e

pytestmark = pytest.mark.gpu

SMALL = dict(layers=3, hidden=256, inter=768, heads=4, kv_heads=2, vocab=500, batch=2, seq=96,
             lora=None, cache_mode="int8", group=128, outlier_ratio=0.0)


def _batch(device):
    ids = e2e.random_batch(SMALL, device, seed=4)
    labels = torch.full_like(ids, -100)
    labels[:, :-1] = ids[:, 1:]
    labels[0, :7] = -100
    return ids, labels


def _grads(model, loss):
    loss.backward()
    out = {k: p.grad.detach().clone() for k, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    return out


def test_rotation_and_scores_follow_the_models_own(device):
    """A policy loss with an entropy bonus through the fused forward, and through the
    model's own modules and elementary operations: loss, scores and gradients."""
    model = e2e.build_llama(SMALL, device, dtype=torch.float32, seed=3)
    ids, labels = _batch(device)
    live = labels != -100
    adv = torch.randn(labels.shape, device=device, generator=torch.Generator(device).manual_seed(1))
    # the elementary side: float32 products, torch's math attention
    logits = model(input_ids=ids, use_cache=False).logits
    lp = torch.log_softmax(logits, -1)
    nll = torch.where(live, lp.gather(-1, labels.clamp(min=0)[..., None])[..., 0], 0.0)
    h = torch.where(live, -(lp.exp() * lp).sum(-1), 0.0)
    want_loss = -(adv * nll).sum() - 0.01 * h.sum()
    want = _grads(model, want_loss)
    got_logits = D.forward(model, ids, rope=True)
    assert (got_logits - logits).norm() <= 1e-4 * logits.norm()
    got_lp, got_h, *_ = cpt.token_scores(got_logits, labels, inplace=True)
    assert (got_lp - nll).norm() <= 1e-4 * nll.norm()
    assert (got_h - h).norm() <= 1e-4 * h.norm()
    loss = -(adv * got_lp).sum() - 0.01 * got_h.sum()
    got = _grads(model, loss)
    assert set(got) == set(want)
    for k in want:
        assert (got[k] - want[k]).norm() <= 1e-4 * want[k].norm(), k


def test_score(device):
    model = e2e.build_llama(SMALL, device, dtype=torch.bfloat16, seed=3).eval()
    ids, labels = _batch(device)
    r = D.score(model, ids, labels, top_k=5, temperature=0.9, rope=True)
    with torch.no_grad(), e2e.fused_attention_only():
        logits = D.forward(model, ids, rope=True)
    want = cpt.token_logprobs(logits, labels, top_k=5, temperature=0.9)
    for a, b in zip(r, want):
        assert (a is None and b is None) or torch.equal(a, b)
    assert (r.top_indices[labels == -100] == -1).all()
    assert (r.top_logprobs[..., 0] >= r.logprobs)[labels != -100].all()


@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_steps(device, state):
    """Three distillation steps with the rotation and AdamW: parameters move by what the
    optimizer's formula makes of the step's own gradients."""
    model, _ = e2e.prepare(SMALL, device, seed=3)
    teacher = e2e.build_llama(SMALL, device, seed=5)
    ids, labels = _batch(device)
    top, idx, lse = D.teacher_top(teacher, ids, 20, 2.0)
    opt = cpt.AdamW(model.parameters(), lr=1e-3, weight_decay=0.01, state=state, master=True,
                    max_norm=1.0)
    for step in range(3):
        before = [p.detach().clone() for p in model.parameters()]
        loss = D.train_step(model, opt, ids, labels, top, idx, lse, rope=True)
        assert bool(loss.isfinite()) and bool(opt.norm.isfinite())
        for p, old in zip(model.parameters(), before):
            s = opt.state[p]
            assert s["step"] == step + 1 and p.grad is None
            assert torch.equal(p, s["master"].to(p.dtype))
            # |m / sqrt(v)| of bias-corrected moments is at most sqrt((1 - b1) / (1 - b2) t)
            # of any sequence: 18 here; the fp32 copy moves by lr times that and decay, p by
            # two roundings of it more
            move = (p.float() - old.float()).abs()
            assert (move <= 1e-3 * 18 + (1e-5 + 2.0 ** -7) * old.float().abs()).all()
        if step == 0:
            # the first step's update is lr times the gradient's sign where that is not 0
            moved = torch.cat([(p.float() - o.float()).abs().flatten()
                               for p, o in zip(model.parameters(), before)])
            assert moved.max() > 0


def test_command(device, capsys):
    D.main(["--layers", "1", "--steps", "1", "--warmup", "1", "--rope", "--optimizer", "adamw8bit",
            "--max-norm", "1.0"])
    out = capsys.readouterr().out
    assert "ms a step" in out and "entropy" in out
    with pytest.raises(AssertionError):
        D.main(["--stock", "--rope"])
    with pytest.raises(AssertionError):
        D.main(["--max-norm", "1.0"])
