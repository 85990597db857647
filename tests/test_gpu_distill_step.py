"""The distillation step on a small LLaMA: forward, loss and gradients of the
fused operators against the same model's own modules and elementary torch
operations, in float32 (the attention and GEMMs are the same calls, so the two
differ by fp32 rounding alone: 1e-4 of a tensor's norm) and a bf16 step with
FlashFFN v3 in every MLP."""

import pytest
import torch

from compact_amd import distill_step as D
from compact_amd import e2e

pytestmark = pytest.mark.gpu

SMALL = dict(layers=3, hidden=256, inter=768, heads=4, kv_heads=2, vocab=500, batch=2, seq=96,
             lora=None, cache_mode="int8", group=128, outlier_ratio=0.0)


def _batch(cfg, device):
    ids = e2e.random_batch(cfg, device, seed=4)
    labels = torch.full_like(ids, -100)
    labels[:, :-1] = ids[:, 1:]
    labels[0, :7] = -100
    return ids, labels


def _grads(model, loss):
    loss.backward()
    out = {k: p.grad.detach().clone() for k, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    return out


@pytest.mark.parametrize("tied", [False, True])
def test_matches_the_stock_step(device, tied):
    model = e2e.build_llama(SMALL, device, dtype=torch.float32, seed=3)
    if tied:
        model.lm_head.weight = model.model.embed_tokens.weight
    teacher = e2e.build_llama(SMALL, device, dtype=torch.float32, seed=5)
    ids, labels = _batch(SMALL, device)
    with torch.no_grad():      # float32 attention: torch's math path
        top, idx = teacher(input_ids=ids, use_cache=False).logits.topk(20, dim=-1)
    stock = model(input_ids=ids, use_cache=False).logits
    want_loss = D.stock_loss(stock, top, idx, labels, 2.0, 0.5)
    want = _grads(model, want_loss)
    logits = D.forward(model, ids)
    assert (logits - stock).norm() <= 1e-4 * stock.norm()
    loss = D.distill_loss(logits, top, idx, labels, temperature=2.0, alpha=0.5, inplace=True)
    got = _grads(model, loss)
    assert abs(float(loss) - float(want_loss)) <= 1e-4 * abs(float(want_loss))
    assert set(got) == set(want)
    for k in want:
        assert (got[k] - want[k]).norm() <= 1e-4 * want[k].norm(), k


def test_step_runs_and_learns(device):
    model, opt = e2e.prepare(SMALL, device, seed=3)
    teacher = e2e.build_llama(SMALL, device, seed=5)
    ids, labels = _batch(SMALL, device)
    top, idx, lse = D.teacher_top(teacher, ids, 20, 2.0)
    for group in opt.param_groups:
        group["lr"] = 1e-3
    losses = [float(D.train_step(model, opt, ids, labels, top, idx, lse)) for _ in range(8)]
    assert all(l == l for l in losses) and losses[-1] < losses[0]
