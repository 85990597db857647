"""Further operators of a language model's training step, as they are measured:
the queries' and keys' norms with the position rotation, the given tokens'
log probabilities with entropy and top alternatives, each with its gradient, and
an AdamW step over all of a model's tensors.

A case is a dict of plain values:

op "rope"      direction "forward" / "backward"; `norm` whether heads are normed
               first; `rotary` of `head_dim` columns turn, in pairs of
               neighbours (`interleaved`) or of halves; `fused` whether queries
               and keys are views of one projection's output; positions start
               anywhere below `far`
op "logprobs"  direction "forward" / "backward"; `k` alternatives
op "adamw"     `state` "float32" or "8bit", `master` whether an fp32 copy of the
               parameters is kept, `clip` whether gradients are clipped to their
               global norm; the tensors are a LLaMA's (`rank` 0) or the factors
               of its adapters of that rank on q, v, gate, up and down

8-bit AdamW state: blocks of 128 elements share a power of two 2^s, s one byte
less 134 (255: the block is NaN).  A second moment is E (5 bits) M (3 bits) and
stands for M 2^s (E = 0) or (8 + M) 2^(E - 1 + s), a first moment has a sign and
E of 4 bits; s puts the block's largest value into the top binade.  Values are
rounded up or down at random, in proportion; a nonzero second moment stays so.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100
NORM_EPS = 1e-6
BLOCK = 128
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.95, 1e-8, 0.1
STEP, SEED, MAX_NORM = 100, 12345, 1.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rope(name, direction, batch, seq, heads, kv_heads, head_dim, dtype, norm, rotary=None,
          interleaved=False, fused=False, far=4096):
    return {"name": name, "op": "rope", "direction": direction, "batch": batch, "seq": seq,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "norm": norm, "rotary": rotary or head_dim, "interleaved": interleaved,
            "fused": fused, "far": far}


def _logprobs(name, direction, rows, vocab, k, dtype, temperature):
    return {"name": name, "op": "logprobs", "direction": direction, "rows": rows, "vocab": vocab,
            "k": k, "dtype": dtype, "temperature": temperature}


def _adamw(name, dtype, state, master, clip, layers, hidden, inter, kv, vocab, rank):
    return {"name": name, "op": "adamw", "dtype": dtype, "state": state, "master": master,
            "clip": clip, "layers": layers, "hidden": hidden, "inter": inter, "kv": kv,
            "vocab": vocab, "rank": rank}


def listed():
    return [
        # four sequences' next tokens while a student with normed heads generates: latency
        _rope("rope_4_tokens", "forward", 4, 1, 32, 4, 64, "fp16", True),
        # attention's input in the full fine-tuning step of 8 x 1024 tokens
        _rope("rope_8x1024", "forward", 8, 1024, 32, 4, 64, "bf16", False),
        # normed heads of the 7B step, one projection for q, k and v: backward
        _rope("rope_norm_grad_4x2048", "backward", 4, 2048, 32, 32, 128, "bf16", True, fused=True),
        # a ragged long-context batch in single precision: half of 80 columns turn, by pairs
        _rope("rope_grad_fp32_odd", "backward", 3, 1003, 12, 3, 80, "fp32", True, rotary=40,
              interleaved=True, far=1000000),
        # the sampled tokens of seven answers: latency
        _logprobs("logprobs_7_rows", "forward", 7, 32000, 5, "bf16", 1.0),
        # a policy's half-precision logits, odd vocabulary, temperature 0.7
        _logprobs("logprobs_fp16_odd", "forward", 1531, 50021, 50, "fp16", 0.7),
        # scoring a batch of 8 x 1024 tokens with 20 alternatives each
        _logprobs("logprobs_8192", "forward", 8192, 32000, 20, "bf16", 1.0),
        # the gradient of a policy loss with an entropy bonus over the same batch
        _logprobs("logprobs_grad_8192", "backward", 8192, 32000, 0, "bf16", 1.0),
        # one layer's rank-8 adapters in single precision: latency
        _adamw("adamw_lora_1_layer", "fp32", "float32", False, False, 1, 2048, 5632, 256, 0, 8),
        # 320 adapter factors of the 7B LoRA step, clipped
        _adamw("adamw_lora_32_layers", "bf16", "float32", False, True, 32, 4096, 11008, 4096, 0,
               16),
        # a few layers with embedding and head, moments in 8 bits
        _adamw("adamw_8bit_6_layers", "bf16", "8bit", False, False, 6, 2048, 5632, 256, 32000, 0),
        # full fine-tuning of the 1.1B student: clipped, fp32 copy of the weights
        _adamw("adamw_22_layers", "bf16", "float32", True, True, 22, 2048, 5632, 256, 32000, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["rope", "logprobs", "adamw"])
    direction = rng.choice(["forward", "backward"])
    if op == "rope":
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 2 * rng.randint(4, 150)])
        rotary = head_dim if rng.random() < 0.7 else max(2, head_dim // 4 * 2)
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 7])
        rows = _log_int(rng, 1, max(1, (1 << 26) // ((heads + kv_heads) * head_dim)))
        batch = min(rows, rng.choice([1, 2, 3, 8]))
        return _rope(None, direction, batch, max(1, rows // batch), heads, kv_heads, head_dim,
                     dtype, rng.random() < 0.6, rotary, rng.random() < 0.3, rng.random() < 0.4,
                     _log_int(rng, 16, 1000000))
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 160000)
        if rng.random() < 0.6:
            vocab = max(1024, vocab // 64 * 64)
        rows = _log_int(rng, 1, (1 << 27) // vocab)
        k = rng.choice([0, 1, 5, 20, _log_int(rng, 1, 128)]) if direction == "forward" else 0
        return _logprobs(None, direction, rows, vocab, k, dtype, rng.choice([1.0, 0.7, 1.3]))
    hidden = _log_int(rng, 64, 4096)
    if rng.random() < 0.6:
        hidden = max(64, hidden // 64 * 64)
    inter = int(hidden * rng.uniform(1.5, 4))
    kv = max(1, hidden // rng.choice([1, 2, 4, 8]))
    rank = rng.choice([0, 4, 8, 16])
    vocab = 0 if rank else _log_int(rng, 500, 32000)
    layer = 5 * rank * (hidden + inter) if rank else 4 * hidden * hidden + 3 * hidden * inter
    layers = _log_int(rng, 1, min(32, max(1, (1 << 27) // layer)))
    state = rng.choice(["float32", "8bit"])
    return _adamw(None, dtype, state, dtype != "fp32" and rng.random() < 0.5, rng.random() < 0.5,
                  layers, hidden, inter, kv, vocab, rank)


def _shapes(case):
    """The sizes of the tensors that an AdamW case steps, in the model's order."""
    h, i, kv, r = case["hidden"], case["inter"], case["kv"], case["rank"]
    if r:
        return [n * r for n in (h, h, h, kv, h, i, h, i, i, h)] * case["layers"]
    layer = [h * h, kv * h, kv * h, h * h, i * h, i * h, h * i, h, h]
    return [case["vocab"] * h] + layer * case["layers"] + [h, case["vocab"] * h]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    return {"rope": _prepare_rope, "logprobs": _prepare_logprobs,
            "adamw": _prepare_adamw}[case["op"]](case, dev, gen, DTYPES[case["dtype"]])


def _heads(case, dev, gen, dt):
    """Queries and keys [B, S, H, D] as the projections leave them: some channels
    are ten times as large."""
    b, s, h, hk, d = (case[n] for n in ("batch", "seq", "heads", "kv_heads", "head_dim"))
    if case["fused"]:
        qkv = torch.randn(b, s, h + 2 * hk, d, device=dev, generator=gen)
        qkv[..., ::16] *= 10
        qkv = qkv.to(dt)
        return qkv[:, :, :h], qkv[:, :, h:h + hk]
    q = torch.randn(b, s, h, d, device=dev, generator=gen)
    k = torch.randn(b, s, hk, d, device=dev, generator=gen)
    q[..., ::16] *= 10
    k[..., ::16] *= 10
    return q.to(dt), k.to(dt)


def _prepare_rope(case, dev, gen, dt):
    b, n, d, r = case["batch"], case["seq"], case["head_dim"], case["rotary"]
    s = {"case": case}
    s["q"], s["k"] = _heads(case, dev, gen, dt)
    # a batch's sequences start at positions of their own
    start = torch.randint(0, max(1, case["far"] - n), (b, 1), device=dev, generator=gen)
    s["positions"] = start + torch.arange(n, device=dev)
    s["inv_freq"] = (10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64)
                                 / r)).float()
    s["w_q"] = s["w_k"] = None
    if case["norm"]:
        s["w_q"], s["w_k"] = ((1 + 0.1 * torch.randn(d, device=dev, generator=gen)).to(dt)
                              for _ in range(2))
    if case["direction"] == "backward":
        s["d_q"], s["d_k"] = (torch.randn(t.shape, device=dev, generator=gen).to(dt)
                              for t in (s["q"], s["k"]))
    return s


def _prepare_logprobs(case, dev, gen, dt):
    n, v = case["rows"], case["vocab"]
    s = {"case": case}
    # a spread vocabulary and a few candidates that stand out
    z = torch.randn(n, v, device=dev, generator=gen).mul_(2.0)
    c = min(24, v)
    cand = torch.randint(0, v, (n, c), device=dev, generator=gen)
    z.scatter_add_(1, cand, 4 + 8 * torch.rand(n, c, device=dev, generator=gen))
    s["logits"] = z.to(dt)
    targets = cand[:, 0].clone()
    targets[torch.rand(n, device=dev, generator=gen) < 0.15] = IGNORE   # prompt and padding
    targets[0] = cand[0, 0]
    s["targets"] = targets
    if case["direction"] == "backward":
        # what the forward left, and a policy loss's gradients for it
        log_p = torch.log_softmax(s["logits"].float() / case["temperature"], 1)
        s["lse"] = torch.logsumexp(s["logits"].float() / case["temperature"], 1)
        s["entropy"] = -(log_p.exp() * log_p).sum(1)
        s["d_logprobs"] = torch.randn(n, device=dev, generator=gen)
        s["d_entropy"] = -0.01 * torch.rand(n, device=dev, generator=gen)
        if case["dtype"] == "fp32":
            s["d_logprobs"] /= n
            s["d_entropy"] /= n
    return s


def _prepare_adamw(case, dev, gen, dt):
    """All tensors of a kind lie in one buffer, each from a multiple of 128 elements
    on; what is between them is zero and stays so."""
    sizes = _shapes(case)
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += -(-n // BLOCK) * BLOCK
    s = {"case": case, "sizes": sizes, "at": at}
    live = torch.ones(total, dtype=torch.bool, device=dev)
    for a, n in zip(at, sizes):
        live[a + n:a + -(-n // BLOCK) * BLOCK] = False

    def draw_flat(make):
        return make(torch.randn(total, device=dev, generator=gen)).mul_(live)

    p = draw_flat(lambda t: t.mul_(0.02))
    # gradients of very different sizes, as layers and channels have them
    wide = torch.repeat_interleave(
        torch.randn(-(-total // BLOCK), device=dev, generator=gen).mul_(1.5).exp_(), BLOCK)[:total]
    g = draw_flat(lambda t: t.mul_(wide).mul_(1e-3))
    m = draw_flat(lambda t: t.mul_(wide).mul_(3e-4))
    v = draw_flat(lambda t: t.mul_(wide).mul_(1e-3).square_().add_(m.square()))
    del wide
    # half precision trains under loss scaling
    s["grad_scale"] = 1.0
    if case["dtype"] == "fp16":
        g *= 1024
        s["grad_scale"] = 1 / 1024
    s["p"], s["g"] = p.to(dt), g.to(dt)
    s["master"] = p if case["master"] else None
    if case["state"] == "8bit":
        dither = torch.full((total,), 0.5, device=dev, dtype=torch.float64)
        s["m"], s["m_scale"] = _encode(m, dither, 4)
        s["v"], s["v_scale"] = _encode(v, dither, 5)
    else:
        s["m"], s["v"] = m, v

    def cut(t, unit=1):
        return [t[a // unit:a // unit + -(-n // unit)] for a, n in zip(at, sizes)]

    s["lists"] = {"p": cut(s["p"]), "g": cut(s["g"]), "m": cut(s["m"]), "v": cut(s["v"])}
    if case["master"]:
        s["lists"]["master"] = cut(p)
    if case["state"] == "8bit":
        s["lists"]["m_scale"] = cut(s["m_scale"], BLOCK)
        s["lists"]["v_scale"] = cut(s["v_scale"], BLOCK)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "rope":
        return (_plain_rope if case["direction"] == "forward" else _plain_rope_backward)(s, case)
    if case["op"] == "logprobs":
        return (_plain_logprobs if case["direction"] == "forward"
                else _plain_logprobs_backward)(s, case)
    return _plain_adamw(s, case)


def _run_own(s, case):
    import compact_amd as cpt
    if case["op"] == "rope":
        kw = dict(w_q=s["w_q"], w_k=s["w_k"], eps=NORM_EPS, interleaved=case["interleaved"])
        if case["direction"] == "forward":
            q, k = cpt.qk_rope(s["q"], s["k"], s["positions"], s["inv_freq"], **kw)
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = cpt.qk_rope_backward(s["d_q"], s["d_k"], s["q"], s["k"],
                                                s["positions"], s["inv_freq"], **kw)
        out = {"d_q": dq, "d_k": dk}
        if case["norm"]:
            out["d_w_q"], out["d_w_k"] = dwq, dwk
        return out
    if case["op"] == "logprobs":
        if case["direction"] == "forward":
            r = cpt.token_logprobs(s["logits"], s["targets"], temperature=case["temperature"],
                                   top_k=case["k"], ignore_index=IGNORE)
            out = {"logprobs": r.logprobs, "entropy": r.entropy, "lse": r.lse}
            if case["k"]:
                out["top_logprobs"], out["top_indices"] = r.top_logprobs, r.top_indices
            return out
        return {"d_logits": cpt.token_logprobs_backward(
            s["logits"], s["targets"], s["lse"], s["entropy"], s["d_logprobs"], s["d_entropy"],
            temperature=case["temperature"], ignore_index=IGNORE)}
    t = s["lists"]
    norm = cpt.adamw_step(t["p"], t["g"], t["m"], t["v"], STEP, lr=LR, betas=(BETA1, BETA2),
                          eps=EPS, weight_decay=DECAY, m_scales=t.get("m_scale"),
                          v_scales=t.get("v_scale"), masters=t.get("master"),
                          grad_scale=s["grad_scale"], max_norm=MAX_NORM if case["clip"] else None,
                          seed=SEED)
    out = {"p": s["p"], "m": s["m"], "v": s["v"]}
    if case["state"] == "8bit":
        (out["m"],), (out["v"],) = cpt.adamw_8bit_values([s["m"]], [s["v"]], [s["m_scale"]],
                                                         [s["v_scale"]])
    if case["master"]:
        out["master"] = s["master"]
    if case["clip"]:
        out["norm"] = norm
    return out


def _turn(x, cos, sin, interleaved):
    """The columns of x [..., R] turned by pairs; cos and sin [..., R / 2]."""
    if interleaved:
        a, b = x[..., ::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _angles(s):
    """cos and sin [B, S, 1, R / 2] in fp32: far positions' angles need 64 bits."""
    angle = s["positions"].double()[..., None, None] * s["inv_freq"].double()
    return angle.cos().float(), angle.sin().float()


def _plain_rope(s, case):
    cos, sin = _angles(s)
    r = case["rotary"]
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS) \
                * s["w_" + name].float()
        x = torch.cat([_turn(x[..., :r], cos, sin, case["interleaved"]), x[..., r:]], -1)
        out[name] = x.to(s[name].dtype)
    return out


def _plain_rope_backward(s, case):
    cos, sin = _angles(s)
    r = case["rotary"]
    out = {}
    for name in ("q", "k"):
        d = s["d_" + name].float()
        d = torch.cat([_turn(d[..., :r], cos, -sin, case["interleaved"]), d[..., r:]], -1)
        if case["norm"]:
            x, w = s[name].float(), s["w_" + name].float()
            rho = torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS)
            n = x * rho
            out["d_w_" + name] = (d * n).sum((0, 1, 2)).to(s["w_" + name].dtype)
            d = d * w
            d = rho * (d - n * (d * n).mean(-1, keepdim=True))
        out["d_" + name] = d.to(s["d_" + name].dtype)
    return out


def _log_softmax(s, case):
    t = s["logits"].float()
    t = (t - t.amax(1, keepdim=True)) / case["temperature"]
    return t - t.exp().sum(1, keepdim=True).log()


def _plain_logprobs(s, case):
    z, tau, y = s["logits"].float(), case["temperature"], s["targets"]
    live = (y >= 0) & (y < case["vocab"])
    log_p = _log_softmax(s, case)
    top = z.amax(1)
    out = {"logprobs": torch.where(live, log_p.gather(1, torch.where(live, y, 0)[:, None])[:, 0],
                                   0.0),
           "entropy": torch.where(live, -(log_p.exp() * log_p).sum(1), 0.0),
           "lse": torch.where(live, top / tau + ((z - top[:, None]) / tau).exp().sum(1).log(),
                              0.0)}
    if case["k"]:
        # whole numbers that sort as (value, lower index first)
        bits = (z + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, -1 - (bits & 0x7FFFFFFF), bits) << 32
        key += 0xFFFFFFFF - torch.arange(case["vocab"], device=z.device)
        idx = 0xFFFFFFFF - (torch.topk(key, case["k"], dim=1).values & 0xFFFFFFFF)
        out["top_logprobs"] = torch.where(live[:, None], log_p.gather(1, idx), -math.inf)
        out["top_indices"] = torch.where(live[:, None], idx, -1)
    return out


def _plain_logprobs_backward(s, case):
    y, tau = s["targets"], case["temperature"]
    live = (y >= 0) & (y < case["vocab"])
    log_p = s["logits"].float() / tau - s["lse"][:, None]
    p = log_p.exp()
    d = -p * (s["d_logprobs"][:, None] + s["d_entropy"][:, None] * (log_p + s["entropy"][:, None]))
    d = d.scatter_add(1, torch.where(live, y, 0)[:, None], s["d_logprobs"][:, None])
    return {"d_logits": (d * (live / tau)[:, None]).to(s["logits"].dtype)}


def _mix(h):
    """A 32-bit number (in int64) whose bits each depend on all of h's."""
    h = h ^ (h >> 16)
    h = (h * 0x243F6A89) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x1E3779B1) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _dither(s, total):
    """Two numbers in [0, 1) an element, of 16 bits each, from (seed, step, the
    tensor's place in the list, the element's place in the tensor)."""
    dev = s["p"].device
    starts = torch.tensor(s["at"] + [total], device=dev)
    i = torch.arange(len(s["at"]), device=dev)
    key = _mix((SEED * 0x37E15163 + STEP * 0x6A09E667 + i * 0x3C6EF373) & 0xFFFFFFFF)
    key = torch.repeat_interleave(key - starts[:-1] * 0x1E3779B9, starts.diff())
    r = _mix((key + torch.arange(total, device=dev) * 0x1E3779B9) & 0xFFFFFFFF)
    return (r & 0xFFFF).double() / 65536, (r >> 16).double() / 65536


def _pow2(n):
    """2^n in 64 bits, exactly."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _encode(x, dither, ebits):
    """(codes, scale bytes) of x in blocks, a step's fraction rounded by `dither`; in
    64 bits, which hold a scaled value and its dither's sum as they are."""
    blocks = x.double().view(-1, BLOCK)
    top = blocks.abs().amax(1)
    s = (torch.frexp(top).exponent - 1 - ((1 << ebits) + 1)).clamp(min=-133)
    s = torch.where(top > 0, s, -133)
    y = blocks.abs() * _pow2(-s)[:, None]
    e = (torch.frexp(y).exponent - 4).clamp(min=0)          # a step is 2^e
    mag = torch.floor(y * _pow2(-e) + dither.view(-1, BLOCK)).int()
    # (8 + M) 2^(E - 1) has E = e + 1, its carry to 16 the next E with M = 0
    code = torch.where(mag >= 8, (e + 1) * 8 + mag - 8, mag).clamp(max=(8 << ebits) - 1)
    if ebits == 5:
        code = torch.where(blocks > 0, code.clamp(min=1), code)
    else:
        code = code | torch.where(blocks < 0, 128, 0)
    return code.to(torch.uint8).view(-1), (s + 134).to(torch.uint8)


def _decode(codes, scales, ebits):
    c = codes.view(-1, BLOCK).int()
    mag = c & ((8 << ebits) - 1)
    e = mag >> 3
    y = torch.where(e > 0, 8 + (mag & 7), mag)
    y = y * _pow2((e - 1).clamp(min=0) + scales.int()[:, None] - 134)
    return (torch.where(c >= 128, -y, y) if ebits == 4 else y).float().view(-1)


def _plain_adamw(s, case):
    g = s["g"].float() * s["grad_scale"]
    out = {}
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        out["norm"] = norm
    bits = case["state"] == "8bit"
    m = _decode(s["m"], s["m_scale"], 4) if bits else s["m"]
    v = _decode(s["v"], s["v_scale"], 5) if bits else s["v"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    p = s["master"] if case["master"] else s["p"].float()
    p = p * (1 - LR * DECAY) - LR / (1 - BETA1 ** STEP) * m / \
        ((v / (1 - BETA2 ** STEP)).sqrt() + EPS)
    if bits:
        dm, dv = _dither(s, g.numel())
        for name, x, d, e in (("m", m, dm, 4), ("v", v, dv, 5)):
            code, scale = _encode(x, d, e)
            s[name].copy_(code)
            s[name + "_scale"].copy_(scale)
            out[name] = _decode(code, scale, e).to(torch.bfloat16)
    else:
        out["m"], out["v"] = s["m"].copy_(m), s["v"].copy_(v)
    if case["master"]:
        out["master"] = s["master"].copy_(p)
    out["p"] = s["p"].copy_(p)
    return out


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s, case)
    if case["op"] == "logprobs":
        return _exact_logprobs(s, case)
    return _exact_adamw(s, case)


def _exact_rope(s, case):
    """Pairs as complex numbers times e^(i angle); the backward is the
    vector-Jacobian product that autograd takes of it."""
    r, h = case["rotary"], case["rotary"] // 2
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=s["q"].device),
                       s["positions"].double()[:, :, None, None] * s["inv_freq"].double())

    def forward(x, w):
        if w is not None:
            x = w * x / (x.square().mean(-1, keepdim=True) + NORM_EPS).sqrt()
        part = x[..., :r]
        a, b = (part[..., ::2], part[..., 1::2]) if case["interleaved"] \
            else (part[..., :h], part[..., h:])
        c = torch.complex(a, b) * unit
        turned = torch.view_as_real(c)
        turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
        return torch.cat([turned, x[..., r:]], -1)

    out = {}
    for n in ("q", "k"):
        x = s[n].double().requires_grad_(True)
        w = None if s["w_" + n] is None else s["w_" + n].double().requires_grad_(True)
        y = forward(x, w)
        if case["direction"] == "forward":
            out[n] = y.detach()
            continue
        grads = torch.autograd.grad(y, [x] if w is None else [x, w], s["d_" + n].double())
        out["d_" + n] = grads[0]
        if w is not None:
            out["d_w_" + n] = grads[1]
    return out


def _exact_logprobs(s, case):
    n, v, tau = case["rows"], case["vocab"], case["temperature"]
    step = max(1, (1 << 25) // v)
    parts = []
    for i in range(0, n, step):
        z, y = s["logits"][i:i + step].double(), s["targets"][i:i + step]
        live = y != IGNORE
        hot = torch.nn.functional.one_hot(y.clamp(min=0), v).double()
        lq = torch.log_softmax(z / tau, 1)
        if case["direction"] == "backward":
            # lse and entropy as the forward left them
            lq = z / tau - s["lse"][i:i + step, None].double()
            a = s["d_logprobs"][i:i + step, None].double()
            b = s["d_entropy"][i:i + step, None].double()
            h = s["entropy"][i:i + step, None].double()
            d = a * (hot - lq.exp()) - b * lq.exp() * (lq + h)
            parts.append({"d_logits": torch.where(live[:, None], d / tau, 0.0)})
            continue
        row = {"logprobs": torch.where(live, (lq * hot).sum(1), 0.0),
               "entropy": torch.where(live, torch.special.entr(lq.exp()).sum(1), 0.0),
               "lse": torch.where(live, torch.logsumexp(z / tau, 1), 0.0)}
        if case["k"]:
            row["top_logprobs"] = torch.where(live[:, None], lq.topk(case["k"], 1).values,
                                              -math.inf)
        parts.append(row)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_adamw(s, case):
    if s["p"].numel() > 1 << 31:
        return None
    bits = case["state"] == "8bit"
    g = s["g"].double() * s["grad_scale"]
    out = {}
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g *= min(1.0, MAX_NORM / (float(out["norm"]) + 1e-6))

    def moment(name, ebits):
        if not bits:
            return s[name].double()
        c = s[name].long()
        e, f = c >> 3 & ((1 << ebits) - 1), (c & 7).double()
        y = torch.where(e > 0, (f + 8) * torch.exp2(e.double() - 1), f)
        y = y * torch.exp2(s[name + "_scale"].double() - 134).repeat_interleave(BLOCK)
        return torch.where(c >> 7 == 1, -y, y) if ebits == 4 else y

    m = torch.lerp(g, moment("m", 4), BETA1)
    v = torch.lerp(g.square(), moment("v", 5), BETA2)
    p = (s["master"] if case["master"] else s["p"]).double()
    p = p - LR * DECAY * p
    p -= LR * (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + EPS)
    if bits:
        def store(x, u, ebits):
            blocks = x.view(-1, BLOCK)
            top = torch.log2(blocks.abs().amax(1, keepdim=True)).floor()
            scale = torch.exp2((top - (1 << ebits) - 1).clamp(min=-133))
            y = blocks.abs() / scale
            unit = torch.exp2((torch.log2(y).floor() - 3).clamp(min=0))
            q = torch.floor(y / unit + u.double().view(-1, BLOCK)) * unit
            if ebits == 5:
                q = torch.where(y > 0, q.clamp(min=1), q)
            q = q.clamp(max=15.0 * 2 ** ((1 << ebits) - 2))
            return torch.where(blocks < 0, -q, q).mul_(scale).view(-1)
        dm, dv = _dither(s, g.numel())
        m, v = store(m, dm, 4), store(v, dv, 5)
    out.update(p=p, m=m, v=v)
    if case["master"]:
        out["master"] = p
    return out


# ---------------------------------------------------------------------------
# the work that a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rope":
        rows = case["batch"] * case["seq"]
        n = rows * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        moved = 3 if case["direction"] == "backward" and case["norm"] else 2
        weights = 2 * case["head_dim"] * e * (moved - 1) if case["norm"] else 0
        flops = 3 + (4 if case["norm"] else 0) + (6 if moved == 3 else 0)
        return {"bytes": moved * n * e + 8 * rows + 2 * case["rotary"] + weights,
                "flops": flops * n}
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["k"]
        # an ignored row is not read; its gradient is written all the same
        read = n * 0.85 if n > 8 else n
        if case["direction"] == "forward":
            return {"bytes": int(read * v * e) + n * (20 + 12 * k), "flops": int(read * v * 6)}
        return {"bytes": int(read * v * e) + n * v * e + 24 * n, "flops": int(read * v * 7)}
    n = sum(_shapes(case))
    per = 3 * e                                             # gradient, parameter in and out
    if case["master"]:
        per = 2 * e + 8                                     # the copy is read in its place
    per += 16 if case["state"] == "float32" else 4 + 4 / BLOCK + 4 + 2   # and the values returned
    return {"bytes": int(n * per) + (4 if case["clip"] else 0), "flops": n * 15}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(c, work(c))
