"""The operators of a language model's training step around its FFN, as they
are measured: embedding lookup with its gradient, the residual norm between
blocks with its gradient, and the distillation loss with its gradient.

A case is a dict of plain values:

op "embedding"      direction "forward" / "backward"
op "residual_norm"  direction "forward" / "backward"; `gate` "none",
                    "channel" ([D]), "sequence" ([B, 1, D]) or "token"
                    ([B, S, 1]); `post` whether the block's output is normed
op "distill"        `grad` False (evaluation: each row's loss) or True
                    (training: their mean and the logits' gradient); `tail`
                    whether the teacher's log-sum-exp over the whole
                    vocabulary is at hand; `hard` whether labels carry a loss

Activations are N(0, 1) streams with a few large channels, token ids follow
Zipf's law with a share of padding, logits are peaked as a trained model's.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100
EPS = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _embedding(name, direction, tokens, vocab, width, dtype):
    return {"name": name, "op": "embedding", "direction": direction, "tokens": tokens,
            "vocab": vocab, "width": width, "dtype": dtype}


def _norm(name, direction, batch, seq, width, dtype, gate, post):
    return {"name": name, "op": "residual_norm", "direction": direction, "batch": batch,
            "seq": seq, "width": width, "dtype": dtype, "gate": gate, "post": post}


def _distill(name, rows, vocab, k, dtype, temperature, grad, hard, tail):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype,
            "temperature": temperature, "grad": grad, "hard": hard, "tail": tail}


def listed():
    return [
        # four sequences' next tokens while the student generates: latency
        _embedding("embed_4_tokens", "forward", 4, 32000, 4096, "bf16"),
        # the embedding of one full fine-tuning batch of 8 x 1024 tokens
        _embedding("embed_8192", "forward", 8192, 32000, 2048, "bf16"),
        # its gradient: a dense table, most of whose rows no token touches
        _embedding("embed_grad_8192", "backward", 8192, 32000, 2048, "bf16"),
        # single-precision gradient of a long ragged batch into a small odd table
        _embedding("embed_grad_fp32_odd", "backward", 20011, 5003, 1001, "fp32"),
        # four next tokens between two blocks: latency
        _norm("norm_4_tokens", "forward", 4, 1, 4096, "fp16", "none", False),
        # between two blocks of the full fine-tuning step, sandwich norms, LayerScale gate
        _norm("norm_8x1024", "forward", 8, 1024, 2048, "bf16", "channel", True),
        # the same in the 7B step's backward
        _norm("norm_grad_4x2048", "backward", 4, 2048, 4096, "bf16", "channel", True),
        # a ragged single-precision batch whose tokens are gated one by one
        _norm("norm_grad_fp32_odd", "backward", 3, 1003, 1999, "fp32", "token", True),
        # a handful of answer tokens distilled online: latency
        _distill("distill_7_rows", 7, 32000, 16, "bf16", 2.0, True, True, False),
        # validation loss against stored teacher logits
        _distill("distill_eval_fp32", 1024, 32000, 64, "fp32", 1.0, False, False, False),
        # half precision under loss scaling, odd vocabulary, teacher's tail known
        _distill("distill_fp16_odd_tail", 1531, 50021, 50, "fp16", 1.5, True, True, True),
        # the distillation step's loss of a whole batch of 8 x 1024 tokens
        _distill("distill_8192", 8192, 32000, 64, "bf16", 2.0, True, True, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["embedding", "residual_norm", "distill"])
    if op == "embedding":
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        # the output (a table, or its rows) no larger than 128 Mi elements
        vocab = _log_int(rng, 500, min(160000, (1 << 27) // width))
        tokens = _log_int(rng, 1, min(100000, (1 << 27) // width))
        return _embedding(None, rng.choice(["forward", "backward"]), tokens, vocab, width, dtype)
    if op == "residual_norm":
        width = _log_int(rng, 64, 8192)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        rows = _log_int(rng, 1, min(100000, (1 << 26) // width))
        batch = rng.choice([1, 2, 3, 4, 8])
        seq = max(1, rows // batch)
        return _norm(None, rng.choice(["forward", "backward"]), batch, seq, width, dtype,
                     rng.choice(["none", "channel", "sequence", "token"]), rng.random() < 0.7)
    vocab = _log_int(rng, 1000, 160000)
    if rng.random() < 0.6:
        vocab = max(1024, vocab // 64 * 64)
    rows = _log_int(rng, 1, (1 << 27) // vocab)
    hard = rng.random() < 0.6
    return _distill(None, rows, vocab, _log_int(rng, 1, 256), dtype,
                    rng.choice([1.0, 1.5, 2.0, 4.0]), rng.random() < 0.7, hard,
                    rng.random() < 0.3)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _zipf(vocab):
    """Zipf's law (exponent 1) over the ranks of a vocabulary."""
    p = 1.0 / np.arange(1, vocab + 1, dtype=np.float64)
    return p / p.sum()


def _ids(case, gen, dev):
    """Token ids: Zipf by rank, ranks spread over the table, a tenth padding (id 0)."""
    vocab, n = case["vocab"], case["tokens"]
    cdf = torch.from_numpy(np.cumsum(_zipf(vocab))).to(dev)
    u = torch.rand(n, device=dev, generator=gen, dtype=torch.float64)
    rank = torch.searchsorted(cdf, u).clamp_(max=vocab - 1)
    ids = torch.randperm(vocab, device=dev, generator=gen)[rank]
    if n > 8:
        ids = torch.where(torch.rand(n, device=dev, generator=gen) < 0.1,
                          torch.zeros_like(ids), ids)
    return ids


def _stream(shape, gen, dev, dtype):
    """An activation stream: N(0, 1), one channel in 256 twenty times as large."""
    t = torch.randn(*shape, device=dev, generator=gen)
    t[..., ::256] *= 20
    return t.to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "embedding":
        s["ids"] = _ids(case, gen, dev)
        s["scale"] = math.sqrt(case["width"])
        if case["direction"] == "forward":
            s["weight"] = (0.02 * torch.randn(case["vocab"], case["width"], device=dev,
                                              generator=gen)).to(dt)
        else:
            s["grad"] = torch.randn(case["tokens"], case["width"], device=dev,
                                    generator=gen).to(dt)
        return s
    if case["op"] == "residual_norm":
        b, n, d = case["batch"], case["seq"], case["width"]
        s["y"] = _stream((b, n, d), gen, dev, dt)
        s["w_pre"] = (1 + 0.1 * torch.randn(d, device=dev, generator=gen)).to(dt)
        s["w_post"] = (1 + 0.1 * torch.randn(d, device=dev, generator=gen)).to(dt) \
            if case["post"] else None
        shape = {"none": None, "channel": (d,), "sequence": (b, 1, d),
                 "token": (b, n, 1)}[case["gate"]]
        s["gate"] = None if shape is None else \
            (0.5 * torch.randn(*shape, device=dev, generator=gen)).to(dt)
        s["scale"], s["residual_scale"] = 0.7, 1.0
        res = _stream((b, n, d), gen, dev, dt)
        if case["direction"] == "forward":
            s["residual"] = res
            return s
        # what the forward left: the residual stream after the block and both norms' scales
        s["residual_out"] = res
        stats = torch.ones(2, b * n, device=dev)
        if case["post"]:
            stats[0] = torch.rsqrt(s["y"].float().pow(2).mean(-1) + EPS).view(-1)
        stats[1] = torch.rsqrt(res.float().pow(2).mean(-1) + EPS).view(-1)
        s["stats"] = stats
        s["d_residual_out"] = torch.randn(b, n, d, device=dev, generator=gen).to(dt)
        s["d_x"] = torch.randn(b, n, d, device=dev, generator=gen).to(dt)
        return s
    n, v, k = case["rows"], case["vocab"], case["k"]
    # both models' logits: a spread vocabulary and a few candidates that stand out
    z = torch.randn(n, v, device=dev, generator=gen).mul_(2.0)
    c = min(24, v)
    cand = torch.randint(0, v, (n, c), device=dev, generator=gen)
    lift = 4 + 8 * torch.rand(n, c, device=dev, generator=gen)
    z.scatter_add_(1, cand, lift)
    teacher = torch.randn(n, v, device=dev, generator=gen)
    teacher.add_(z, alpha=0.7)
    tau = case["temperature"]
    top, idx = torch.topk(teacher, min(k, v), dim=1)
    s["logits"] = z.to(dt)
    s["top_logits"], s["top_indices"] = top, idx.to(torch.int32)
    s["top_lse"] = torch.logsumexp(teacher / tau, 1) if case["tail"] else None
    labels = cand[:, 0].clone()
    labels[torch.rand(n, device=dev, generator=gen) < 0.15] = IGNORE   # prompt and padding
    labels[0] = cand[0, 0]
    s["labels"] = labels
    s["alpha"] = 0.6 if case["hard"] else 1.0
    # half precision trains under loss scaling
    s["grad_out"] = 65536.0 if case["dtype"] == "fp16" else 1.0
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "embedding":
        return _plain_embedding(s, case)
    if case["op"] == "residual_norm":
        return (_plain_norm if case["direction"] == "forward" else _plain_norm_backward)(s)
    return _plain_distill(s, case)


def _run_own(s, case):
    import compact_amd as cpt
    if case["op"] == "embedding":
        if case["direction"] == "forward":
            return {"out": cpt.embedding(s["ids"], s["weight"], s["scale"])}
        return {"d_weight": cpt.embedding_backward(s["grad"], s["ids"], case["vocab"], s["scale"],
                                                   padding_idx=0)}
    if case["op"] == "residual_norm":
        if case["direction"] == "forward":
            r, x, stats = cpt.residual_norm(s["residual"], s["y"], s["w_pre"], w_post=s["w_post"],
                                            gate=s["gate"], scale=s["scale"],
                                            residual_scale=s["residual_scale"], eps=EPS)
            return {"residual": r, "x": x, "stats": stats}
        dr, dy, dwp, dwq, dg = cpt.residual_norm_backward(
            s["d_residual_out"], s["d_x"], s["residual_out"], s["y"], s["stats"], s["w_pre"],
            w_post=s["w_post"], gate=s["gate"], scale=s["scale"],
            residual_scale=s["residual_scale"])
        out = {"d_residual": dr, "d_y": dy, "d_w_pre": dwp}
        if dwq is not None:
            out["d_w_post"] = dwq
        if dg is not None:
            out["d_gate"] = dg
        return out
    loss, grad = cpt.distill_topk(s["logits"], s["top_logits"], s["top_indices"], s["labels"],
                                  top_lse=s["top_lse"], temperature=case["temperature"],
                                  alpha=s["alpha"], ignore_index=IGNORE,
                                  reduction="mean" if case["grad"] else "none",
                                  grad_out=s["grad_out"], want_grad=case["grad"])
    return {"loss": loss, "d_logits": grad} if case["grad"] else {"loss": loss}


def _plain_embedding(s, case):
    if case["direction"] == "forward":
        return {"out": (s["weight"][s["ids"]].float() * s["scale"]).to(s["weight"].dtype)}
    g = s["grad"].float() * s["scale"]
    g = g * (s["ids"] != 0).unsqueeze(1)
    d = torch.zeros(case["vocab"], case["width"], device=g.device)
    d.index_add_(0, s["ids"], g)
    return {"d_weight": d.to(s["grad"].dtype)}


def _plain_norm(s):
    dt = s["y"].dtype
    y, u = s["y"].float(), s["y"].float()
    rho1 = torch.ones(y.shape[:-1] + (1,), device=y.device)
    if s["w_post"] is not None:
        rho1 = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        u = y * rho1 * s["w_post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    r = s["residual_scale"] * s["residual"].float() + s["scale"] * u
    rho2 = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    x = r * rho2 * s["w_pre"].float()
    return {"residual": r.to(dt), "x": x.to(dt),
            "stats": torch.stack([rho1.reshape(-1), rho2.reshape(-1)])}


def _sum_to(t, shape):
    """The sum of t over the axes along which a tensor of `shape` was broadcast."""
    while t.dim() > len(shape):
        t = t.sum(0)
    for i, n in enumerate(shape):
        if n == 1 and t.shape[i] != 1:
            t = t.sum(i, keepdim=True)
    return t


def _plain_norm_backward(s):
    dt = s["y"].dtype
    y, r = s["y"].float(), s["residual_out"].float()
    dr, dx = s["d_residual_out"].float(), s["d_x"].float()
    rho1 = s["stats"][0].view(*y.shape[:-1], 1)
    rho2 = s["stats"][1].view(*y.shape[:-1], 1)
    n2 = r * rho2
    dn2 = dx * s["w_pre"].float()
    t = dr + rho2 * (dn2 - n2 * (dn2 * n2).mean(-1, keepdim=True))
    out = {"d_residual": (s["residual_scale"] * t).to(dt)}
    gate = None if s["gate"] is None else s["gate"].float()
    du = s["scale"] * t if gate is None else s["scale"] * t * gate
    if s["w_post"] is not None:
        n1 = y * rho1
        u = n1 * s["w_post"].float()
        dn1 = du * s["w_post"].float()
        dy = rho1 * (dn1 - n1 * (dn1 * n1).mean(-1, keepdim=True))
    else:
        u, dy = y, du
    out["d_y"] = dy.to(dt)
    out["d_w_pre"] = (dx * n2).sum((0, 1)).to(dt)
    if s["w_post"] is not None:
        out["d_w_post"] = (du * n1).sum((0, 1)).to(dt)
    if gate is not None:
        out["d_gate"] = _sum_to(s["scale"] * t * u, s["gate"].shape).to(dt)
    return out


def _plain_distill(s, case):
    tau, alpha = case["temperature"], s["alpha"]
    z = s["logits"].float()
    idx = s["top_indices"].long()
    keep = s["labels"] != IGNORE
    scale = 1.0 / keep.sum().clamp(min=1)

    def log_softmax(t):
        t = t - t.amax(1, keepdim=True)
        return t - t.exp().sum(1, keepdim=True).log()

    logq = log_softmax(z / tau)
    if s["top_lse"] is None:
        logp = log_softmax(s["top_logits"].float() / tau)
    else:
        logp = s["top_logits"].float() / tau - s["top_lse"].unsqueeze(1)
    p = logp.exp()
    soft = (p * (logp - logq.gather(1, idx))).sum(1)
    mass = p.sum(1)
    rest = None
    if s["top_lse"] is not None:
        rest = (1 - mass).clamp(min=0)
        others = logq.exp().scatter(1, idx, 0.0).sum(1)
        soft = soft + torch.where(rest > 0, rest * (rest.log() - others.log()), 0.0)
        mass = mass + rest
    loss = alpha * tau * tau * soft
    if case["hard"]:
        logq1 = log_softmax(z)
        y = s["labels"].clamp(min=0).unsqueeze(1)
        loss = loss - (1 - alpha) * logq1.gather(1, y).squeeze(1)
    loss = torch.where(keep, loss, 0.0)
    if not case["grad"]:
        return {"loss": loss}
    out = {"loss": loss.sum() * scale}
    q = logq.exp()
    d = q * mass.unsqueeze(1)
    if rest is not None:
        d = d - (q * (rest / others).unsqueeze(1)).scatter(1, idx, 0.0)
    d = (alpha * tau) * d.scatter_add(1, idx, -p)
    if case["hard"]:
        d = d + (1 - alpha) * logq1.exp()
        d = d.scatter_add(1, y, torch.full_like(y, alpha - 1, dtype=d.dtype))
    d = d * (keep * scale * s["grad_out"]).unsqueeze(1)
    out["d_logits"] = d.to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in s.items()}
    if case["op"] == "embedding":
        return _exact_embedding(s, case)
    if case["op"] == "residual_norm":
        return _exact_norm(s, case)
    return _exact_distill(s, case)


def _exact_embedding(s, case):
    ids, c = s["ids"], s["scale"]
    if case["direction"] == "forward":
        return {"out": torch.nn.functional.embedding(ids, s["weight"]) * c}
    live = ids != 0
    order = torch.argsort(ids[live], stable=True)
    rows, seg = s["grad"][live][order], ids[live][order]
    d = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device=rows.device)
    if seg.numel():
        d.index_put_((seg,), rows * c, accumulate=True)
    return {"d_weight": d}


def _exact_norm(s, case):
    """The forward as it is defined; the backward as its vector-Jacobian
    product with both norms' scales as the forward left them."""
    d, a, b = case["width"], s["scale"], s["residual_scale"]
    y = s["y"].reshape(-1, d)
    rows = y.shape[0]
    wq = torch.ones(d, dtype=torch.float64, device=y.device) if s["w_post"] is None \
        else s["w_post"]
    g = torch.ones(rows, d, dtype=torch.float64, device=y.device) if s["gate"] is None \
        else s["gate"].expand(case["batch"], case["seq"], d).reshape(rows, d)
    if case["direction"] == "forward":
        rho1 = torch.ones(rows, dtype=torch.float64, device=y.device)
        if s["w_post"] is not None:
            rho1 = (y.square().sum(1) / d + EPS).pow(-0.5)
        r = b * s["residual"].reshape(-1, d) + a * g * (y * rho1[:, None] * wq)
        rho2 = (r.square().sum(1) / d + EPS).pow(-0.5)
        shape = s["y"].shape
        return {"residual": r.view(shape), "x": (r * rho2[:, None] * s["w_pre"]).view(shape),
                "stats": torch.stack((rho1, rho2))}
    rho1, rho2 = s["stats"][0][:, None], s["stats"][1][:, None]
    dx = s["d_x"].reshape(-1, d)
    n1, n2 = y * rho1, s["residual_out"].reshape(-1, d) * rho2
    v = dx * s["w_pre"]
    t = s["d_residual_out"].reshape(-1, d) \
        + rho2 * (v - n2 * ((v * n2).sum(1, keepdim=True) / d))
    w = a * g * t * wq
    dy = rho1 * (w - n1 * ((w * n1).sum(1, keepdim=True) / d)) if s["w_post"] is not None else w
    out = {"d_residual": (b * t).view(s["y"].shape), "d_y": dy.view(s["y"].shape),
           "d_w_pre": (dx * n2).sum(0)}
    if s["w_post"] is not None:
        out["d_w_post"] = (a * g * t * n1).sum(0)
    if s["gate"] is not None:
        dg = (a * t * n1 * wq).view(case["batch"], case["seq"], d)
        out["d_gate"] = {"channel": lambda: dg.sum((0, 1)),
                         "sequence": lambda: dg.sum(1, keepdim=True),
                         "token": lambda: dg.sum(2, keepdim=True)}[case["gate"]]()
    return out


def _exact_distill(s, case):
    """Row blocks at a time: the loss and gradient over the vocabulary, with
    the teacher laid out as a dense row."""
    tau, alpha, n = case["temperature"], s["alpha"], case["rows"]
    labels, idx = s["labels"], s["top_indices"].long()
    count = max(1, int((labels != IGNORE).sum()))
    step = max(1, (1 << 25) // case["vocab"])
    losses, grads = [], []
    for i in range(0, n, step):
        z, y, j = s["logits"][i:i + step], labels[i:i + step], idx[i:i + step]
        keep = (y != IGNORE).double()
        lq = torch.log_softmax(z / tau, 1)
        t = s["top_logits"][i:i + step] / tau
        lp = torch.log_softmax(t, 1) if s["top_lse"] is None \
            else t - s["top_lse"][i:i + step, None]
        p = torch.zeros_like(z).scatter_(1, j, lp.exp())
        loss = (lp.exp() * (lp - lq.gather(1, j))).sum(1)
        d = lq.exp() * p.sum(1, keepdim=True) - p
        if s["top_lse"] is not None:
            rest = (1 - p.sum(1)).clamp(min=0)
            out = torch.ones_like(z).scatter_(1, j, 0.0)
            lo = torch.logsumexp(lq.masked_fill(out == 0, -math.inf), 1)
            loss = loss + torch.special.xlogy(rest, rest) - torch.where(rest > 0, rest * lo, 0.0)
            d = d + rest[:, None] * (lq.exp() - out * (lq - lo[:, None]).exp())
        loss, d = alpha * tau ** 2 * loss, alpha * tau * d
        if case["hard"]:
            l1 = torch.log_softmax(z, 1)
            yy = y.clamp(min=0)[:, None]
            loss = loss - (1 - alpha) * l1.gather(1, yy)[:, 0]
            d = d + (1 - alpha) * (l1.exp() - torch.zeros_like(z).scatter_(1, yy, 1.0))
        losses.append(loss * keep)
        if case["grad"]:
            grads.append(d * (keep * s["grad_out"] / count)[:, None])
    losses = torch.cat(losses)
    return {"loss": losses.sum() / count, "d_logits": torch.cat(grads)} if case["grad"] \
        else {"loss": losses}


# ---------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------

def _distinct(case):
    """The expected number of distinct ids among the tokens, padding too."""
    p = _zipf(case["vocab"])
    n = case["tokens"] if case["tokens"] <= 8 else 0.9 * case["tokens"]
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "embedding":
        n, d, v = case["tokens"], case["width"], case["vocab"]
        if case["direction"] == "forward":
            return {"bytes": 8 * n + int(_distinct(case) * d * e) + n * d * e, "flops": n * d}
        # padding's rows are not needed
        live = n if n <= 8 else 0.9 * n
        return {"bytes": 8 * n + int(live * d * e) + v * d * e, "flops": int(2 * live * d)}
    if case["op"] == "residual_norm":
        n, d = case["batch"] * case["seq"], case["width"]
        gate = {"none": 0, "channel": d, "sequence": case["batch"] * d, "token": n}[case["gate"]]
        params = (d + (d if case["post"] else 0) + gate) * e
        if case["direction"] == "forward":
            return {"bytes": 4 * n * d * e + params + 8 * n, "flops": 10 * n * d}
        return {"bytes": 6 * n * d * e + 2 * params + 8 * n, "flops": 24 * n * d}
    n, v, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
    # an ignored row is not read; its gradient is written all the same
    read = n * 0.85 if n > 8 else n
    softmaxes = 2 if case["hard"] and case["temperature"] != 1 else 1
    nbytes = int(read * (v * e + 8 * k)) + 8 * n + (4 * n if case["tail"] else 0)
    nbytes += 4 if case["grad"] else 4 * n
    flops = int(read * v * (1 + 3 * softmaxes))
    if case["grad"]:
        nbytes += n * v * e
        flops += int(read * v * (1 + 3 * softmaxes))
    return {"bytes": nbytes, "flops": flops}
