"""How the sequence operators sit in autograd: what is changed between forward
and backward is seen, by the host glue and by the Python paths."""
import pytest
import torch

import seq_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["glue", "python"])
def path(request, monkeypatch):
    from flash_cqt import _seq_native
    if request.param == "python":
        monkeypatch.setattr(_seq_native, "load_glue", lambda: None)
    return request.param


@pytest.mark.parametrize("which", ["positions", "freq"])
def test_positions_changed_before_the_backward_pass(path, which):
    """They are needed again, so a change in place raises; one after it, or
    without gradients, does not."""
    from flash_cqt import sequence
    q = torch.randn(2, 5, 2, 16, device="cuda", requires_grad=True)
    pos, freq = torch.rand(5, 1, device="cuda") * 9, sequence.rotary_frequencies((8,))
    changed = pos if which == "positions" else freq
    y, _ = sequence.head_norm_rotary(q, q, pos, freq, (8,))
    changed.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    y, _ = sequence.head_norm_rotary(q, q, pos, freq, (8,))
    y.square().sum().backward()
    changed.add_(1)
    with torch.no_grad():
        sequence.head_norm_rotary(q, q, pos, freq, (8,))
        changed.add_(1)


def test_positions_of_other_kinds(path):
    """Whole numbers, a view, values made in inference mode, values with a
    gradient of their own: the same gradients, none of them for positions."""
    from flash_cqt import sequence
    x = torch.randn(2, 5, 2, 16, device="cuda")
    freq = sequence.rotary_frequencies((8,))
    whole = torch.tensor([[3], [1], [4], [1], [5]], device="cuda")
    with torch.inference_mode():
        inferred = whole.float()
    leaf = whole.float().requires_grad_(True)
    found = []
    for pos in (whole, whole.float(), torch.stack([whole.float()] * 3)[1], inferred, leaf):
        q = x.clone().requires_grad_(True)
        y, z = sequence.head_norm_rotary(q, q, pos, freq, (8,))
        ((y * x).sum() + z.sum()).backward()
        found.append(q.grad)
        if pos is whole:
            whole += 0                                                       # converted: a copy of its own was kept
    assert leaf.grad is None and all(torch.equal(found[0], g) for g in found[1:])
    wide = x.cpu().double().requires_grad_(True)
    angle = ref.angles(whole.cpu().expand(2, 5, 1), freq.cpu(), (8,))
    y = ref.head_norm_rotary(wide, None, angle, 1e-6, False)
    ((y * wide.detach()).sum() + y.sum()).backward()
    ref.close(found[0], wide.grad, slack=2)


def test_forward_mode_is_refused(path):
    """Tangents of any input raise, by dual tensors and by torch.func; so do its other transforms."""
    import torch.autograd.forward_ad as fwd
    from flash_cqt import sequence
    x = torch.randn(2, 3, 2, 16, device="cuda")
    w, pos, freq = torch.ones(16, device="cuda"), torch.rand(3, 1, device="cuda"), sequence.rotary_frequencies((8,))
    g, S = -torch.rand(2, device="cuda"), torch.randn(2, 2, 16, 16, device="cuda")
    calls = [(lambda q, k, w, p, f: sequence.head_norm_rotary(q, k, p, f, (8,), w)[0], (x, x, w, pos, freq)),
             (lambda q, k, v, g, S: sequence.decay_attention(q, k, v, g, state=S)[0], (x, x, x, g, S)),
             (lambda q, k, v, g, S: sequence.decay_attention_step(q, k, v, g, S), (x[:, 0], x[:, 0], x[:, 0], g, S.clone()))]
    for call, args in calls:
        call(*args)
        for i in range(len(args)):
            for leaf in (False, True):
                with fwd.dual_level():
                    t = args[i].clone().requires_grad_(leaf and call is not calls[2][0])
                    with pytest.raises(NotImplementedError):
                        call(*args[:i], fwd.make_dual(t, torch.ones_like(t)), *args[i + 1:])
            with pytest.raises(RuntimeError):                                # NotImplementedError among them
                torch.func.jvp(lambda t: call(*args[:i], t, *args[i + 1:]), (args[i],), (torch.ones_like(args[i]),))
        with fwd.dual_level():
            call(*args)
        for transform in (torch.func.vmap, lambda f: torch.func.grad(lambda t: f(t).sum())):
            with pytest.raises((RuntimeError, ValueError)):
                transform(lambda t: call(t, *args[1:]))(args[0][None].expand(3, *args[0].shape) if transform is torch.func.vmap else args[0])
    from flash_cqt import optim
    p, m = torch.ones(4, device="cuda"), torch.zeros(4, device="cuda")
    with fwd.dual_level():
        for i in range(2):
            t = [fwd.make_dual(p.clone(), p.clone()) if i == j else p.clone() for j in range(2)]
            with pytest.raises(NotImplementedError):
                optim.adamw_step([t[0]], [t[1]], [m], [m.clone()], step=1, lr=0.1)
    assert not m.any()


def at_odd_place(t, by=3):
    """The same values in a contiguous view that starts at no multiple of 16 bytes."""
    flat = torch.cat([t.new_zeros(by), t.flatten()])
    return flat[by:].view(t.shape)


@pytest.mark.parametrize("T", [5, 700])                                      # one segment, and several
def test_states_at_any_place(path, T):
    """A first state in a view at an odd place, and the gradient of a last state
    that was joined behind three numbers, which autograd hands over as such a
    view: the bits of those at other places."""
    from flash_cqt import sequence
    gen = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(2, T, 2, 16, device="cuda", generator=gen) for _ in range(3))
    g, S = -torch.rand(2, device="cuda", generator=gen), torch.randn(2, 2, 16, 16, device="cuda", generator=gen)
    more, weight = torch.zeros(3, device="cuda"), torch.randn(2 * 2 * 16 * 16, device="cuda", generator=gen)
    found = []
    for odd in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, g, S)]
        first = at_odd_place(leaves[4]) if odd else leaves[4]
        assert (first.data_ptr() % 16 != 0) == odd
        o, last = sequence.decay_attention(*leaves[:4], state=first)
        joined = torch.cat([more, last.flatten()])[3:] if odd else last.flatten()
        found.append([o, last, *torch.autograd.grad((joined * weight).sum() + o.sum(), leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*found))
    with torch.no_grad():
        _, last = sequence.decay_attention(q, k, v, g, state=at_odd_place(S, 1))
    assert torch.equal(last, found[0][1])


def spread(t):
    """The same values, elements of the last dimension (of a vector, its own) two places apart."""
    return t.new_empty(*t.shape, 2)[..., 0].copy_(t)


def test_saved_tensors_with_other_strides(path):
    """Hooks may give saved tensors back laid out differently: the same gradients.
    Another type, or another shape, raises."""
    from flash_cqt import sequence
    gen = torch.Generator("cuda").manual_seed(6)
    q, k, v = (torch.randn(2, 700, h, 16, device="cuda", generator=gen) for h in (4, 2, 2))
    w, g, S = (torch.rand(*s, device="cuda", generator=gen) for s in ((16,), (2,), (2, 2, 16, 16)))
    pos, freq = torch.rand(2, 700, 1, device="cuda", generator=gen) * 9, sequence.rotary_frequencies((8,))
    lengths = torch.tensor([700, 333], dtype=torch.int32, device="cuda")

    def run(unpack):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, w, -g, S)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            a, b = sequence.head_norm_rotary(leaves[0], leaves[1], pos, freq, (8,), leaves[3], leaves[3])
            o, last = sequence.decay_attention(a, b, leaves[2], leaves[4], state=leaves[5], lengths=lengths)
        return torch.autograd.grad((o, last), leaves, (o.detach(), last.detach()))
    want = run(lambda t: t)
    for unpack in (spread, at_odd_place, lambda t: spread(t.clone())):
        assert all(torch.equal(x, y) for x, y in zip(want, run(unpack)))
    for unpack in (lambda t: t.half() if t.is_floating_point() else t, lambda t: t[..., :8], lambda t: t.cpu()):
        with pytest.raises(RuntimeError, match="saved tensor"):
            run(unpack)
