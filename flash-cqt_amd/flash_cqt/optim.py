"""AdamW over many tensors at once, on one kernel (libflashcqt_seq.so).

    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)
    loss.backward()
    opt.step()

A CQT layer's learnt gains and a small model's weights are dozens of small
tensors: an elementwise launch for each of a step's operations on each of them
takes far longer than their arithmetic. Here a launch serves up to 56 tensors.
With state_bits=8 the moments take one byte an element and one float32 scale
for every 256, instead of four bytes; codes are drawn between a value's two
neighbours, so that moments follow AdamW's rule over many steps.
"""
import math
import operator

import torch

from . import _seq_native as _n

__all__ = ["AdamW", "adamw_step", "read_moments"]


_ORDINARY = frozenset((torch.Tensor, torch.nn.Parameter))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _blocks(n):
    return -(-n // _n.ADAMW_BLOCK)


def _tensor(name, t, like, dtypes):
    if not (torch.is_tensor(t) and t.is_cuda and t.is_contiguous() and t.dtype in dtypes):
        raise ValueError(f"{name} must be a contiguous tensor on a GPU of a type among {[str(d) for d in dtypes]}")
    if t.device != like.device or t.numel() != like.numel():
        raise ValueError(f"{name} {tuple(t.shape)} on {t.device} does not match {tuple(like.shape)} on {like.device}")
    return t.data_ptr()


def _scale(name, t, like):
    if not (torch.is_tensor(t) and t.dtype == torch.float32 and t.is_contiguous() and t.device == like.device
            and t.numel() == _blocks(like.numel())):
        raise ValueError(f"{name} must be a contiguous float32 tensor of {_blocks(like.numel())} elements beside its tensor")
    return t.data_ptr()


def _clipping(grad_scale, devices):
    if grad_scale is None:
        return
    if not (torch.is_tensor(grad_scale) and grad_scale.is_cuda and grad_scale.numel() == 1 and grad_scale.dtype == torch.float32):
        raise ValueError("grad_scale must be a float32 tensor of one element on the GPU")
    for d in devices:
        if grad_scale.device != d:
            raise ValueError(f"grad_scale is on {grad_scale.device}, a tensor on {d}")


def _factors(step, lr, betas, eps, weight_decay):
    b1, b2 = betas
    if not (step >= 1 and lr >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1 and eps > 0 and weight_decay >= 0):
        raise ValueError(f"step {step}, lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}: "
                         "out of their ranges (step >= 1, lr and weight_decay >= 0, 0 <= betas < 1, eps > 0)")
    return (b1, 1 - b1, b2, 1 - b2, 1 - lr * weight_decay, lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step), eps)


def _scale_lists(scales, count):
    if scales is None:
        return None
    ms, vs = scales
    if len(ms) != count or len(vs) != count:
        raise ValueError("scales: a list for the first and one for the second moments, as long as the others")
    return ms, vs


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               scales=None, grad_scale=None, seed=None):
    """One AdamW step (decoupled weight decay) of the tensors `params`, in place.

    params, grads: contiguous tensors of float32, bfloat16 or float16 on one
    GPU, a gradient of its tensor's type. exp_avgs, exp_avg_sqs: their moments,
    float32 tensors; or, with scales=(list, list), uint8 codes of as many
    elements, with a float32 scale for every 256 of them (read_moments gives
    the values they stand for; zeros in both are moments of zero). step counts
    from 1. grad_scale: a float32 tensor of one element on the GPU that every
    gradient is multiplied by first (a clipping factor), or None.

    16-bit tensors are computed in float32 and rounded once, to the nearest."""
    count = len(params)
    if not len(grads) == len(exp_avgs) == len(exp_avg_sqs) == count:
        raise ValueError("params, grads, exp_avgs and exp_avg_sqs differ in length")
    f = _factors(step, lr, betas, eps, weight_decay)
    lists = _scale_lists(scales, count)
    if seed is not None:
        seed = operator.index(seed)
        if not 0 <= seed < 1 << 64:
            raise ValueError(f"seed is {seed}: 0 to 2^64 - 1 wanted")
    at = 0 if seed is None else operator.index(step)
    glue = None if torch.compiler.is_compiling() else _n.load_glue()
    if glue is not None and all(
            _ORDINARY.issuperset(map(type, ts)) for ts in (params, grads, exp_avgs, exp_avg_sqs, *(lists or ()))):
        ms, vs = lists or ((), ())
        if glue.adamw(params, grads, exp_avgs, exp_avg_sqs, ms, vs, lists is not None, f, grad_scale, seed, at):
            return
    _n.no_tangents(*params, *grads, *exp_avgs, *exp_avg_sqs, grad_scale)
    bits = 32 if lists is None else 8
    state = (torch.float32,) if bits == 32 else (torch.uint8,)
    _clipping(grad_scale, ())
    groups = {}
    for i, p in enumerate(params):
        d = _n.AdamwTensor(_tensor(f"params[{i}]", p, p, _n.DTYPES), _tensor(f"grads[{i}]", grads[i], p, (p.dtype,)),
                           _tensor(f"exp_avgs[{i}]", exp_avgs[i], p, state),
                           _tensor(f"exp_avg_sqs[{i}]", exp_avg_sqs[i], p, state),
                           None if lists is None else _scale(f"scales[0][{i}]", lists[0][i], p),
                           None if lists is None else _scale(f"scales[1][{i}]", lists[1][i], p), p.numel())
        groups.setdefault((p.dtype, p.device), []).append(d)
    _clipping(grad_scale, {device for _, device in groups})
    for i, ((dtype, device), ds) in enumerate(groups.items()):
        ts, gs, stream = (_n.AdamwTensor * len(ds))(*ds), _ptr(grad_scale), _n.stream_handle(device.index)
        if bits == 8 and seed is not None:
            status = _n.load().fcqt_adamw_drawn(ts, len(ds), _n.DTYPES[dtype], _n.AdamwFactors(*f), gs,
                                                (seed + (i << 48)) % (1 << 64), at, stream)
        else:
            status = _n.load().fcqt_adamw(ts, len(ds), _n.DTYPES[dtype], bits, _n.AdamwFactors(*f), gs, stream)
        _n.check(status, "adamw_step")
    torch.autograd.graph.increment_version([*params, *exp_avgs, *exp_avg_sqs, *(x for xs in lists or () for x in xs)])


def read_moments(exp_avgs, exp_avg_sqs, scales, *, out=None):
    """The values that 8-bit moments stand for: two lists of float32 tensors
    (new ones, or the contiguous ones of out=(list, list))."""
    count = len(exp_avgs)
    if len(exp_avg_sqs) != count:
        raise ValueError("exp_avgs and exp_avg_sqs differ in length")
    ms, vs = _scale_lists(scales, count)
    if out is None:
        out = tuple([torch.empty(m.shape, dtype=torch.float32, device=m.device) for m in exp_avgs] for _ in range(2))
    elif len(out[0]) != count or len(out[1]) != count:
        raise ValueError("out: two lists as long as the moments")
    glue = None if torch.compiler.is_compiling() else _n.load_glue()
    if glue is not None and all(_ORDINARY.issuperset(map(type, ts)) for ts in (exp_avgs, exp_avg_sqs, ms, vs, *out)) \
            and glue.read(exp_avgs, exp_avg_sqs, ms, vs, *out):
        return out
    groups = {}
    for i, m in enumerate(exp_avgs):
        d = _n.AdamwTensor(_tensor(f"out[0][{i}]", out[0][i], m, (torch.float32,)),
                           _tensor(f"out[1][{i}]", out[1][i], m, (torch.float32,)),
                           _tensor(f"exp_avgs[{i}]", m, m, (torch.uint8,)),
                           _tensor(f"exp_avg_sqs[{i}]", exp_avg_sqs[i], m, (torch.uint8,)),
                           _scale(f"scales[0][{i}]", ms[i], m), _scale(f"scales[1][{i}]", vs[i], m), m.numel())
        groups.setdefault(m.device, []).append(d)
    for device, ds in groups.items():
        _n.check(_n.load().fcqt_adamw_read((_n.AdamwTensor * len(ds))(*ds), len(ds), _n.stream_handle(device.index)),
                 "read_moments")
    torch.autograd.graph.increment_version([*out[0], *out[1]])
    return out


class AdamW(torch.optim.Optimizer):
    """torch.optim's interface over adamw_step: parameter groups, schedulers,
    state_dict; parameters are contiguous. state_bits: 32, or 8 for one byte a
    moment (decided when a parameter first steps; tensors under min_8bit
    elements keep 32 bits). seed: of the draws that 8-bit moments are rounded by (adamw_step); runs of
    one seed and the same gradients are the same."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit=4096,
                 seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is {state_bits}: 8 or 32 wanted")
        if not 0 <= operator.index(seed) < 1 << 32:
            raise ValueError(f"seed is {seed}: 0 to 2^32 - 1 wanted")
        _factors(1, lr, betas, eps, weight_decay)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit=min_8bit, seed=seed))

    def _state(self, p, group):
        """The state of p, a new one where it has none (not yet kept)."""
        s = self.state.get(p)
        if not s:
            s = {"step": 0}
            eight = group["state_bits"] == 8 and p.numel() >= group["min_8bit"]
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros(p.shape, dtype=torch.uint8 if eight else torch.float32, device=p.device)
                if eight:
                    s[name + "_scale"] = torch.zeros(_blocks(p.numel()), dtype=torch.float32, device=p.device)
        return s

    def load_state_dict(self, state_dict):
        """As torch.optim's, which casts a state to its parameter's type: codes
        and scales keep theirs. One of torch.optim.AdamW's is taken up too, its
        moments as float32."""
        for group in state_dict["param_groups"]:
            for name, other in (("amsgrad", True), ("maximize", True), ("decoupled_weight_decay", False)):
                if group.get(name) is other:
                    raise ValueError(f"the state is one of {name}={other}, which this AdamW does not do")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            for name, x in self.defaults.items():
                group.setdefault(name, x)
        index = {i: p for g, h in zip(state_dict["param_groups"], self.param_groups)
                 for i, p in zip(g["params"], h["params"])}
        for i, s in state_dict["state"].items():
            p = index[i]
            for name, x in s.items():
                if name == "step":
                    self.state[p][name] = int(x)
                elif torch.is_tensor(x):
                    x = x.detach().clone().to(p.device)
                    self.state[p][name] = x.float().contiguous() if x.is_floating_point() else x

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step under stream capture would replay one step's factors; capture adamw_step "
                               "only where that is meant")
        # all is looked over before anything changes: a call that raises leaves weights, moments and counts as they were
        calls = []
        for i, group in enumerate(self.param_groups):
            # tensors of one count of steps and one kind of moments go together
            sets = {}
            for j, p in enumerate(group["params"]):
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW takes dense gradients")
                if not (p.is_cuda and p.is_contiguous() and p.dtype in _n.DTYPES):       # (its gradient is alike)
                    _tensor(f"parameter {j} of group {i}", p, p, _n.DTYPES)
                s = self._state(p, group)
                sets.setdefault((s["step"] + 1, "exp_avg_scale" in s), []).append((p, p.grad.contiguous(), s))
            for (step, eight), ps in sets.items():
                _factors(step, group["lr"], group["betas"], group["eps"], group["weight_decay"])
                _clipping(grad_scale, {p.device for p, _, _ in ps})
                calls.append((i, group, step, eight, ps))
        for i, group, step, eight, ps in calls:
            scales = tuple([s[n] for _, _, s in ps] for n in ("exp_avg_scale", "exp_avg_sq_scale")) if eight else None
            adamw_step([p for p, _, _ in ps], [g for _, g, _ in ps], [s["exp_avg"] for _, _, s in ps],
                       [s["exp_avg_sq"] for _, _, s in ps], step=step, lr=group["lr"], betas=group["betas"],
                       eps=group["eps"], weight_decay=group["weight_decay"], scales=scales, grad_scale=grad_scale,
                       seed=group["seed"] + (i << 32))
            for p, _, s in ps:
                s["step"] = step
                self.state[p] = s
        return loss
