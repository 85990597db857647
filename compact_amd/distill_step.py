"""A distillation step of a LLaMA student with every operator outside attention
on the library's kernels: scaled embedding, residual norms between the blocks,
FlashFFN v3 in every MLP, and the loss of a teacher's top logits.

  forward(model, ids)      the student's logits (embedding, norms and adds fused)
  teacher_top(model, ids)  a teacher's top-K logits, their indices and log-sum-exp
  train_step(...)          forward, distill_loss, backward, optimizer

`python -m compact_amd.distill_step` times the step on a random-initialised
student of the TinyLlama configuration of e2e.py (synthetic tokens, a
random-initialised two-layer teacher); `--stock` runs torch's embedding, the
model's own norms and adds, and the loss in elementary operations instead.
Attention, the LM head and AdamW are stock in both.
"""

from __future__ import annotations

import argparse
import time

import torch
import torch.nn.functional as F

from . import e2e
from .lm import EmbeddingFunction, ResidualNormFunction, distill_loss


def forward(model, ids, embed_scale: float = 1.0) -> torch.Tensor:
    """Logits of a LlamaForCausalLM for whole sequences `ids` [B, S]: the model's
    own weights, attention and MLPs; each block's residual add and the norm that
    follows it are one operator."""
    m = model.model
    emb = m.embed_tokens
    h = EmbeddingFunction.apply(ids, emb.weight, embed_scale, emb.padding_idx)
    pos = torch.arange(ids.shape[1], device=ids.device).unsqueeze(0)
    rope = m.rotary_emb(h, position_ids=pos)
    layers = list(m.layers)

    def norm(residual, y, module):
        return ResidualNormFunction.apply(residual, y, module.weight, None, None, 1.0, 1.0,
                                          module.variance_epsilon)

    r, x = norm(h, None, layers[0].input_layernorm)
    for layer, after in zip(layers, [n.input_layernorm for n in layers[1:]] + [m.norm]):
        a = layer.self_attn(x, position_embeddings=rope, attention_mask=None)[0]
        r, x = norm(r, a, layer.post_attention_layernorm)
        r, x = norm(r, layer.mlp(x), after)
    return model.lm_head(x)


@torch.no_grad()
def teacher_top(teacher, ids, k: int, temperature: float):
    """(top logits [B, S, k], indices, log-sum-exp of all logits / temperature)."""
    with e2e.fused_attention_only():
        logits = teacher(input_ids=ids).logits.float()
    top, idx = logits.topk(k, dim=-1)
    return top, idx.int(), torch.logsumexp(logits / temperature, -1)


def stock_loss(logits, top, idx, labels, temperature: float, alpha: float):
    """The loss of distill_loss (no tail) in elementary operations."""
    live = labels != -100
    z = logits.float()
    p = F.softmax(top.float() / temperature, -1)
    logq = F.log_softmax(z / temperature, -1).gather(-1, idx.long())
    soft = temperature ** 2 * (p * (p.clamp(min=1e-30).log() - logq)).sum(-1)
    hard = F.cross_entropy(z.flatten(0, 1), labels.flatten(), reduction="none",
                           ignore_index=-100).view(labels.shape)
    loss = alpha * soft + (1 - alpha) * hard
    return (loss * live).sum() / live.sum().clamp(min=1)


def train_step(model, opt, ids, labels, top, idx, lse=None, *, temperature: float = 2.0,
               alpha: float = 0.5, stock: bool = False) -> torch.Tensor:
    """One step; labels [B, S] are the next tokens (-100: no loss there).  Returns
    the loss."""
    with e2e.fused_attention_only():
        if stock:
            logits = model(input_ids=ids, use_cache=False).logits
            loss = stock_loss(logits, top, idx, labels, temperature, alpha)
        else:
            # the logits are this step's own: their gradient takes their memory
            loss = distill_loss(forward(model, ids), top, idx, labels, top_lse=lse,
                                temperature=temperature, alpha=alpha, inplace=True)
        loss.backward()
    opt.step()
    opt.zero_grad(set_to_none=True)
    return loss.detach()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--stock", action="store_true")
    ap.add_argument("--layers", type=int, default=e2e.CONFIGS["c4"]["layers"])
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--warmup", type=int, default=2)
    ap.add_argument("--k", type=int, default=64)
    ap.add_argument("--tail", action="store_true",
                    help="hold the teacher's mass outside its top k against the student's")
    args = ap.parse_args(argv)
    assert not (args.stock and args.tail), "the stock loss has no tail"
    dev = torch.device("cuda", 0)
    cfg = dict(e2e.CONFIGS["c4"], layers=args.layers)
    model, opt = e2e.prepare(cfg, dev)
    teacher = e2e.build_llama(dict(cfg, layers=2), dev, seed=1).eval()
    ids = e2e.random_batch(cfg, dev)
    labels = torch.full_like(ids, -100)
    labels[:, :-1] = ids[:, 1:]
    top, idx, lse = teacher_top(teacher, ids, args.k, 2.0)
    del teacher
    torch.cuda.reset_peak_memory_stats()
    times = []
    for i in range(args.warmup + args.steps):
        torch.cuda.synchronize()
        t = time.perf_counter()
        loss = train_step(model, opt, ids, labels, top, idx, lse if args.tail else None,
                          stock=args.stock)
        torch.cuda.synchronize()
        if i >= args.warmup:
            times.append((time.perf_counter() - t) * 1e3)
    print(f"{'stock' if args.stock else 'fused'} operators, {args.layers} layers, "
          f"{ids.numel()} tokens: {sorted(times)[len(times) // 2]:.2f} ms a step, peak "
          f"{torch.cuda.max_memory_allocated() / 2 ** 30:.2f} GiB, loss {float(loss):.4f}")


if __name__ == "__main__":
    main()
