"""optim.AdamW's state: a step that is refused changes nothing."""
import copy

import pytest
import torch

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
