"""optim.AdamW's state: a step that is refused changes nothing, and one of
torch.optim.AdamW's is taken up."""
import copy

import pytest
import torch

import seq_ref as ref

pytestmark = pytest.mark.gpu


def same(a, b):
    if torch.is_tensor(a):
        return torch.is_tensor(b) and a.dtype == b.dtype and torch.equal(a, b)
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(map(same, a, b))
    return a == b


@pytest.mark.parametrize("begun", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_step_changes_nothing(bits, begun):
    """A parameter that the kernels cannot take, a wrong factor, a wrong clipping
    factor: weights, moments and counts of all groups stay, and the same step
    done right then gives what it would have given."""
    from flash_cqt import optim
    gen = torch.Generator("cuda").manual_seed(1)
    good = [torch.nn.Parameter(torch.randn(5000, device="cuda", generator=gen)) for _ in range(2)]
    bad = torch.nn.Parameter(torch.randn(8, 6, device="cuda", generator=gen).t())                # not contiguous
    double = torch.nn.Parameter(torch.randn(9, device="cuda", generator=gen).double())
    host = torch.nn.Parameter(torch.randn(9))
    grads = [torch.randn(5000, device="cuda", generator=gen) for _ in good]
    opt = optim.AdamW([dict(params=[good[0], bad]), dict(params=[good[1], double, host])], state_bits=bits)
    for p, g in zip(good, grads):
        p.grad = g
    if begun:
        opt.step()
    before, weights = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in good]

    def refused(error=ValueError, **kw):
        with pytest.raises(error):
            opt.step(**kw)
        assert same(opt.state_dict(), before) and all(torch.equal(p, w) for p, w in zip(good, weights))
    for p in (bad, double, host):
        p.grad = torch.ones_like(p)
        refused()
        p.grad = None
    for scale in (torch.ones(2, device="cuda"), torch.ones(1), torch.ones(1, device="cuda", dtype=torch.float64), 0.5):
        refused(grad_scale=scale)
    opt.param_groups[1]["lr"] = -1.0
    before = copy.deepcopy(opt.state_dict())
    refused()
    opt.param_groups[1]["lr"] = opt.param_groups[0]["lr"]
    opt.step()
    qs = [torch.nn.Parameter(w.clone()) for w in weights]
    other = optim.AdamW([dict(params=[q]) for q in qs], state_bits=bits)
    if begun:
        for i, (p, q) in enumerate(zip(good, qs)):
            other.state[q] = {k: v.clone() if torch.is_tensor(v) else v for k, v in before["state"][2 * i].items()}
    for q, g in zip(qs, grads):
        q.grad = g
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(good, qs))
    assert opt.state[good[0]]["step"] == opt.state[good[1]]["step"] == 1 + begun


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_state_of_torchs_adamw(dtype):
    """Its steps are tensors and its moments of the parameter's type: taken up as
    counts and float32, tensors go in one call, and the run goes on by the rule."""
    from flash_cqt import optim
    gen = torch.Generator("cuda").manual_seed(2)
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).to(dtype)) for n in (40, 7)]
    how = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    theirs = torch.optim.AdamW(ps, **how)
    grads = [[torch.randn(p.shape, device="cuda", generator=gen).to(dtype) for p in ps] for _ in range(3)]
    for gs in grads[:2]:
        for p, g in zip(ps, gs):
            p.grad = g
        theirs.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    ours = optim.AdamW(qs)
    ours.load_state_dict(theirs.state_dict())
    assert ours.param_groups[0]["lr"] == 1e-2 and ours.param_groups[0]["state_bits"] == 32
    calls = []
    step, optim.adamw_step = optim.adamw_step, lambda *a, **k: (calls.append(len(a[0])), step(*a, **k))
    try:
        for q, g in zip(qs, grads[2]):
            q.grad = g
        ours.step()
    finally:
        optim.adamw_step = step
    assert calls == [2] and all(ours.state[q]["step"] == 3 for q in qs)
    for p, q, g in zip(ps, qs, grads[2]):
        s = theirs.state[p]
        want = ref.adamw(p.detach().cpu().double(), g.cpu().double(), s["exp_avg"].cpu().double(), s["exp_avg_sq"].cpu().double(), step=3, **how)
        for x, y, t in zip((q, ours.state[q]["exp_avg"], ours.state[q]["exp_avg_sq"]), want, (dtype, torch.float32, torch.float32)):
            ref.close(x, y, t)
    for kw in (dict(amsgrad=True), dict(maximize=True)):
        before = copy.deepcopy(ours.state_dict())
        with pytest.raises(ValueError, match="does not do"):
            ours.load_state_dict(torch.optim.AdamW(ps, **kw).state_dict())
        assert same(ours.state_dict(), before)
    with pytest.raises(ValueError, match="decoupled"):
        ours.load_state_dict(torch.optim.Adam(ps).state_dict())
