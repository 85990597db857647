"""AdamW over many tensors in few launches, moments in float32 or in 8 bits.

  adamw_step, grad_norm, adamw_8bit_values    AdamW

`adamw_step` steps lists of tensors in place; `AdamW` is the torch optimizer
around it.  Parameters are float32, float16 or bfloat16, gradients of their type or
float32, an fp32 copy of 16-bit parameters optional.  Gradients can be clipped to
their global norm within the step, which costs one more read of them and no
synchronisation.  The reference leaves the optimizer to torch.  There is no CPU
path.

8-bit moments take 2 bytes and 1/64 an element in place of 8.  128 consecutive
elements share a power of two (a byte each for both moments); a code has three
bits of mantissa and four (first moment, signed) or five (second) of exponent, and
values are rounded up or down at random, in proportion, so that averages that
move by less than a code's step a time still move.
"""

from __future__ import annotations

import torch

from . import _lib
from ._lib import check
from .kernels import _guard, _ptr, _require_device, _stream, _timed

BLOCK = 128         # elements of an 8-bit moment that share a scale


def _first(tensors):
    """The device index of a list's first tensor, which the others have to share."""
    dev = tensors[0].get_device()
    if dev < 0:
        _require_device(tensors[0])
    return dev


def _listed(tensors):
    """None, a list or a tuple, or what else is iterable as a list."""
    return tensors if tensors is None or type(tensors) in (list, tuple) else list(tensors)


def _scalar(t, dev, what):
    assert t.dtype == torch.float32 and t.numel() == 1 and t.get_device() == dev, \
        f"{what}: one float32 on the tensors' device expected"
    return t.data_ptr()


def _workspace(like, count, elements):
    nbytes = _lib.api().cpt_adamw_workspace_bytes(count, elements)
    assert nbytes >= 0, f"{count} tensors of {elements} elements: out of range"
    return like.new_empty(nbytes, dtype=torch.uint8)


def grad_norm(grads, *, grad_scale: float = 1.0, out=None) -> torch.Tensor:
    """The 2-norm of grad_scale times all gradients as one vector, a float32 scalar on
    their device; it is summed in 64 bits.  One dtype and device."""
    grads = list(grads)
    assert grads, "grad_norm: no gradients"
    dev = _first(grads)
    table, at, total, _, dt, loose = _lib.lists().grads_table(grads)
    if loose:
        for i in loose:
            grads[i] = grads[i].contiguous()
        table, at, total, _, dt, _ = _lib.lists().grads_table(grads)
    if out is None:
        out = grads[0].new_empty((), dtype=torch.float32)
    out_at = _scalar(out, dev, "out")
    ws = _workspace(grads[0], len(grads), total)
    with _guard(grads[0]), _timed("grad_norm"):
        rc = _lib.api().cpt_grad_norm(dt, at, len(grads), float(grad_scale), out_at, ws.data_ptr(),
                                      _stream(grads[0]))
    check(rc, "grad_norm")
    return out


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, m_scales=None, v_scales=None,
               masters=None, grad_scale: float = 1.0, max_norm: float | None = None, norm=None,
               seed: int = 0):
    """One AdamW step over lists of tensors, in place:

        g = grad * grad_scale * min(1, max_norm / (norm + 1e-6))
        m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
        p = p - lr weight_decay p - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps)

    params: one dtype and device, any dense layout; grads: their dtype or float32 (one
    that lies otherwise than its parameter is copied); exp_avgs, exp_avg_sqs: float32,
    laid out as the parameters.  With m_scales and v_scales (uint8, one a 128 elements)
    the moments are 8-bit codes (uint8 [numel], in the order of the parameter's memory)
    rounded by `seed`.  masters: float32 parameters that are stepped in the place of
    16-bit ones, which become their rounding.  Zeros are a valid start for all moments,
    codes and scales.  What is written lies apart from all else; a gradient may be its
    parameter or moment itself.

    step: this step's number, from 1 (for all, or a list: runs of equal numbers share
    launches), or int64 counts of the steps done on the device (one tensor of
    len(params), or one each), which the call increases: what a captured graph needs.
    lr: a number, or a float32 scalar on the device.

    max_norm clips by the global norm of grad_scale * grads (inf: measures it alone),
    which is returned (float32 scalar on the device; else None); `norm` gives it where it
    is known, as for more tensors than these.  A norm that is not finite leaves
    parameters, moments and counts as they were."""
    params, grads = list(params), list(grads)
    exp_avgs, exp_avg_sqs = _listed(exp_avgs), _listed(exp_avg_sqs)
    m_scales, v_scales, masters = _listed(m_scales), _listed(v_scales), _listed(masters)
    b1, b2 = betas
    assert (m_scales is None) == (v_scales is None), "m_scales and v_scales belong together"
    assert 0 <= b1 < 1 and 0 <= b2 < 1, f"betas={betas}"
    assert eps >= 0 and weight_decay >= 0, f"eps={eps}, weight_decay={weight_decay}"
    assert max_norm is None or max_norm > 0, f"max_norm={max_norm}"
    assert norm is None or max_norm is not None, "norm goes with max_norm"
    if not params:
        assert not grads, "gradients without parameters"
        return norm
    assert grads, "parameters without gradients"
    if not isinstance(step, (int, torch.Tensor)):
        step = _listed(step)
    dev = _first(params)
    lists = _lib.lists()
    args = exp_avgs, exp_avg_sqs, m_scales, v_scales, masters, step, True
    table, at, total, dt, gdt, loose = lists.adamw_table(params, grads, *args)
    if loose:
        for i in loose:
            grads[i] = torch.empty_like(params[i], dtype=grads[i].dtype).copy_(grads[i])
        table, at, total, dt, gdt, _ = lists.adamw_table(params, grads, *args)
    lr_at = norm_at = ws = None
    if isinstance(lr, torch.Tensor):
        lr_at, lr = _scalar(lr, dev, "lr"), 0.0
    assert lr >= 0, f"lr={lr}"
    given, p0, count = norm is not None, params[0], len(params)
    if max_norm is not None:
        if not given:
            norm = p0.new_empty((), dtype=torch.float32)
        norm_at = _scalar(norm, dev, "norm")
    first = step if isinstance(step, (int, torch.Tensor)) else step[0]
    if max_norm is not None or not isinstance(first, int):
        ws = _workspace(p0, count, total)
    with _guard(p0), _timed("adamw_step"):
        rc = _lib.api().cpt_adamw(dt, gdt, int(m_scales is not None), int(masters is not None), at,
                                  count, float(lr), lr_at, float(b1), float(b2), float(eps),
                                  float(weight_decay), float(grad_scale),
                                  0.0 if max_norm is None else float(max_norm), int(given),
                                  seed & 0xFFFFFFFF, norm_at, _ptr(ws), _stream(p0))
    check(rc, "adamw_step")
    # autograd refuses a graph that still needs the old parameters
    lists.bump_versions(params)
    return norm


def adamw_8bit_values(exp_avgs, exp_avg_sqs, m_scales, v_scales):
    """What 8-bit moments stand for: two lists of bfloat16 tensors, shaped as the codes,
    which hold the values exactly (NaN for a block with a value that was not finite)."""
    exp_avgs = list(exp_avgs)
    if not exp_avgs:
        return [], []
    assert m_scales is not None and v_scales is not None, "both moments' scales expected"
    _first(exp_avgs)
    m = [t.new_empty(t.shape, dtype=torch.bfloat16) for t in exp_avgs]
    v = [t.new_empty(t.shape, dtype=torch.bfloat16) for t in exp_avgs]
    table, at, *_ = _lib.lists().adamw_table(m, v, exp_avgs, exp_avg_sqs, m_scales, v_scales, None,
                                             1, False)
    with _guard(m[0]), _timed("adamw_8bit_values"):
        rc = _lib.api().cpt_adamw_8bit_values(at, len(m), _stream(m[0]))
    check(rc, "adamw_8bit_values")
    return m, v


def _check_options(g):
    """A group's options: in range, and no other formula asked for."""
    lr, betas, eps, decay, state = (g[n] for n in ("lr", "betas", "eps", "weight_decay", "state"))
    assert state in ("float32", "8bit"), f"state={state!r}: 'float32' or '8bit' expected"
    assert isinstance(lr, torch.Tensor) or lr >= 0, f"lr={lr}"
    assert 0 <= betas[0] < 1 and 0 <= betas[1] < 1, f"betas={betas}"
    assert eps >= 0 and decay >= 0, f"eps={eps}, weight_decay={decay}"
    for name in ("maximize", "amsgrad"):
        assert not g.get(name), f"AdamW: {name}={g[name]} is not what its step does"
    assert g.get("decoupled_weight_decay", True) or decay == 0, \
        "AdamW: decay within the gradient is not what its step does"


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step by adamw_step.

    state: "float32" or "8bit" moments.  master: keep an fp32 copy of 16-bit
    parameters and step that.  max_norm clips all gradients by their global norm (inf:
    measures it alone); the last step's norm is in `norm` (on the device), and a step
    whose norm is not finite changes nothing (but the step count, which is only known to
    the device where capturable).  seed: of the 8-bit moments' rounding.  capturable: step
    counts on the device, so that a step can be captured into a graph (give lr as a float32
    tensor there to change it); the step before has to be an eager one, which makes the
    state."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state: str = "float32", master: bool = False,
                 max_norm: float | None = None, seed: int = 0, capturable: bool = False):
        assert max_norm is None or max_norm > 0, f"max_norm={max_norm}"
        self.max_norm, self.seed, self.norm = max_norm, seed, None
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state=state,
                        master=master, capturable=capturable)
        _check_options(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _init_state(self, p, group):
        s = self.state[p]
        master = group["master"] and p.dtype != torch.float32
        if s and (not master or "master" in s):
            return s
        _require_device(p)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the state has to be there before a step is captured")
        dev = p.device
        if not s:
            s["step"] = torch.zeros((), dtype=torch.int64, device=dev) if group["capturable"] else 0
            if group["state"] == "8bit":
                n, blocks = p.numel(), -(-p.numel() // BLOCK)
                for name, size in (("exp_avg", n), ("exp_avg_sq", n), ("m_scale", blocks),
                                   ("v_scale", blocks)):
                    s[name] = torch.zeros(size, dtype=torch.uint8, device=dev)
            else:
                s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                s["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        if master:
            s["master"] = p.detach().to(torch.float32, copy=True)
        return s

    @staticmethod
    def _move_counts(params, states, capturable):
        """Step counts, to the device or from it: of a group whose `capturable` was changed."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the counts have to be on the device before a step is "
                               "captured")
        for p, s in zip(params, states):
            if isinstance(s["step"], torch.Tensor if capturable else int):
                continue
            n = int(s["step"])
            s["step"] = torch.tensor(n, device=p.device) if capturable else n

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: float = 1.0):
        """One step over the parameters that have gradients; grad_scale multiplies these
        (the inverse of a loss scale)."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # lists of one kind each: the types, the device, and what the state holds
        buckets = []
        for group in self.param_groups:
            params = group["params"]
            grads = [p.grad for p in params]
            if any([g is None for g in grads]):
                params = [p for p, g in zip(params, grads) if g is not None]
                grads = [g for g in grads if g is not None]
            if not params:
                continue
            states = [self.state[p] for p in params]
            lists = _lib.lists()
            empty, form, counts = lists.state_forms(states)
            if empty or (group["master"] and form < 2):
                for p, s in zip(params, states):
                    if not s or (group["master"] and "master" not in s):
                        self._init_state(p, group)
                _, form, counts = lists.state_forms(states)
            if counts != int(bool(group["capturable"])):
                self._move_counts(params, states, group["capturable"])
            if form >= 0 and lists.one_kind(params) and lists.one_kind(grads):
                buckets.append((group, params, grads, states))
                continue
            kinds = [(p.dtype, g.dtype, p.get_device(), "m_scale" in s, "master" in s)
                     for p, g, s in zip(params, grads, states)]
            for kind in dict.fromkeys(kinds):
                at = [i for i, other in enumerate(kinds) if other == kind]
                buckets.append((group, *([x[i] for i in at] for x in (params, grads, states))))
        norm = None
        if self.max_norm is not None and len(buckets) > 1:
            norms = [grad_norm(grads, grad_scale=grad_scale) for _, _, grads, _ in buckets]
            # in 64 bits as each list's own: the squares of norms past 1e19 are inf in fp32
            norm = grad_norm([n.to(norms[0].device) for n in norms])
        for k, (group, params, grads, states) in enumerate(buckets):
            bits8, master = "m_scale" in states[0], "master" in states[0]
            capturable, steps = group["capturable"], [s["step"] for s in states]
            if not capturable and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a captured step needs capturable=True")
            if not capturable:
                steps = [n + 1 for n in steps]
            got = adamw_step(
                params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                steps, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                weight_decay=group["weight_decay"],
                m_scales=[s["m_scale"] for s in states] if bits8 else None,
                v_scales=[s["v_scale"] for s in states] if bits8 else None,
                masters=[s["master"] for s in states] if master else None,
                grad_scale=grad_scale, max_norm=self.max_norm,
                norm=None if norm is None else norm.to(params[0].device), seed=self.seed + k)
            if not capturable:
                for s, n in zip(states, steps):
                    s["step"] = n
            if norm is None:
                self.norm = got
        if norm is not None:
            self.norm = norm
        return loss

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm, "seed": self.seed,
                "norm": self.norm}

    def load_state_dict(self, state_dict):
        """As torch's, with every part of the state in the type that it was saved in.  A state
        of torch.optim.AdamW is taken too: its moments as float32
        (and the group's `state` with them); the fp32 copy that `master` asks for is then made
        of the parameters by the next step.  One whose options ask for
        another formula (maximize, amsgrad, decay within the gradient) is refused."""
        for g in state_dict["param_groups"]:
            _check_options({**self.defaults, **g})
        before = self.param_groups
        super().load_state_dict(state_dict)
        # what a state of torch's does not say stays as each group has it
        for group, old, saved in zip(self.param_groups, before, state_dict["param_groups"]):
            for name, value in old.items():
                group.setdefault(name, value)
            if "state" not in saved and any(i in state_dict["state"] for i in saved["params"]):
                group["state"] = "float32"      # as the moments that came
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        owners = [(p, g) for g in self.param_groups for p in g["params"]]
        for i, (p, group) in zip(ids, owners):
            saved = state_dict["state"].get(i)
            if saved is None:
                continue
            s = {n: t.detach().to(p.device, copy=True) if isinstance(t, torch.Tensor) else t
                 for n, t in saved.items()}
            for n in ("exp_avg", "exp_avg_sq"):
                if n in s and s[n].is_floating_point():
                    s[n] = s[n].float()
            count = int(s.get("step", 0))
            s["step"] = torch.tensor(count, device=p.device) if group["capturable"] else count
            self.state[p] = s
