"""The distillation step's optimizer against its formula, from the step's own gradients."""

import pytest
import torch

import compact_amd as cpt
from compact_amd import distill_step as D
from compact_amd import e2e
from tests.test_gpu_adamw import _close_param, _moments, _param
from tests.test_gpu_step_path import SMALL, _batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state", ["float32", "8bit"])
def test_steps_follow_the_formula(device, state):
    """Each of three steps: the fp32 copies against the formula in 64 bits at the gradients
    that the step found, clipped by the norm that it gives, from the moments before it."""
    model, _ = e2e.prepare(SMALL, device, seed=3)
    teacher = e2e.build_llama(SMALL, device, seed=5)
    ids, labels = _batch(device)
    top, idx, lse = D.teacher_top(teacher, ids, 20, 2.0)
    hp = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    max_norm = 0.25
    opt = cpt.AdamW(model.parameters(), **hp, state=state, master=True, max_norm=max_norm)
    params = [p for p in model.parameters() if p.requires_grad]
    found = {}

    def before(opt, args, kw):
        for p in params:
            s = opt.state.get(p)
            if not s:
                m = v = torch.zeros(p.shape)
            elif state == "8bit":
                (m,), (v,) = cpt.adamw_8bit_values([s["exp_avg"]], [s["exp_avg_sq"]],
                                                   [s["m_scale"]], [s["v_scale"]])
                m, v = (t.float().cpu().view(p.shape) for t in (m, v))
            else:
                m, v = s["exp_avg"].cpu().clone(), s["exp_avg_sq"].cpu().clone()
            w = s["master"].clone() if s else p.detach().float()
            found[p] = p.grad.cpu().clone(), m, v, w.cpu()

    opt.register_step_pre_hook(before)
    for step in range(3):
        D.train_step(model, opt, ids, labels, top, idx, lse, rope=True)
        norm = opt.norm.cpu()
        want = torch.cat([found[p][0].double().flatten() for p in params]).norm()
        assert abs(float(norm) - float(want)) <= 2.0 ** -23 * float(want)
        clip = (torch.tensor(max_norm) / (norm + 1e-6)).clamp(max=1.0)
        moved = 0
        for p in params:
            g, m, v, w = found[p]
            m1, v1 = _moments(g, m, v, clip=clip, hp=hp)
            want, up = _param(w, m1, v1, step + 1, hp)
            _close_param(opt.state[p]["master"], want, up, torch.float32)
            assert torch.equal(p, opt.state[p]["master"].to(p.dtype))
            moved += int((up.abs() > 0.1 * hp["lr"]).sum())
        assert moved > 0.1 * sum(p.numel() for p in params)
