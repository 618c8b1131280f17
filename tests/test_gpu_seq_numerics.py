"""What the sequence operators' arithmetic keeps where errors can hide behind a
rounding or add up over many tokens or steps."""
import pytest
import torch

import seq_ref as ref

pytestmark = pytest.mark.gpu


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dims", [(128, 128), (64, 64)], ids=str)
def test_16_bit_results_are_32_bit_ones_rounded(dtype, dims):
    """o, dq, dk and dv differ from the float64 values' own rounding only where
    those lie within fp32's error of the place between two numbers.

    With a mean error e and numbers u apart, a value rounds to the other side
    with probability 2 e / u and is then u off: the square of the difference is
    2 e u on average. e is at most FP32 / 4 = 5e-7 of the values' general size
    (sums of some hundreds of terms; 16-bit operands would leave 1.3e-6), and u
    on average 2^-7 / ln 2 / 2 of |x| (from 2^-7 to 2^-8 of it), |x| 0.8 of the
    general size for normal values: 4.5e-3 for bf16, an eighth for fp16."""
    from flash_cqt import sequence
    B, T, Hq, Hk, (Dk, Dv) = 1, 640, 4, 2, dims
    gen = torch.Generator().manual_seed(51)
    q, k = randn(gen, B, T, Hq, Dk, dtype=dtype), randn(gen, B, T, Hk, Dk, dtype=dtype)
    v, go = randn(gen, B, T, Hk, Dv, dtype=dtype), randn(gen, B, T, Hq, Dv, dtype=dtype)
    g = torch.tensor([-0.3, -2.0 ** -8])
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o, _ = sequence.decay_attention(*leaves, g.cuda())
    got = [o, *torch.autograd.grad(o, leaves, go.cuda())]
    wide = [t.double().requires_grad_(True) for t in (q, k, v)]
    w, _ = ref.decay_attention(*wide, g.double(), Dk ** -0.5, None, None)
    want = [w, *torch.autograd.grad(w, wide, go.double())]
    u = 4.5e-3 * ref.HALF_ULP[dtype] / ref.HALF_ULP[torch.bfloat16]
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, want):
        y = y.detach().to(dtype).double()
        rel = ((x.detach().cpu().double() - y).norm() / y.norm()).item()
        assert rel <= (2 * ref.FP32 / 4 * u) ** 0.5, (name, rel)


def recurrence(k, v, g, state):
    """The states after each token in float64: k, v [B, T, H, D]."""
    lam = torch.exp(g.double())[:, None, None]
    for t in range(k.shape[1]):
        state = lam * state + k[:, t].double().unsqueeze(-1) * v[:, t].double().unsqueeze(-2)
        yield state


@pytest.mark.parametrize("pool", [False, True])
def test_single_tokens_add_up_to_the_sequence(pool):
    """6000 single tokens, heads that remember a few to a hundred thousand of
    them. Every token rounds a state twice, by up to 2^-24 of it and to either
    side: over the horizon of 1 / |g| tokens (6000 at most) that is 2^-23 of its
    root. (A decay that is off by the same 2^-25 at each of them would be
    horizon times that: 1.8e-4 for 6000.)"""
    from flash_cqt import sequence
    T, H, D = 6000, 5, 16
    gen = torch.Generator().manual_seed(61)
    q, k, v = (randn(gen, 1, T, H, D).cuda() + 0.3 for _ in range(3))
    g = -torch.tensor([0.7, 0.3, 2.0 ** -10.5, 1e-4, 1e-5], device="cuda")
    S = torch.zeros(3 if pool else 1, H, D, D, device="cuda")
    slots = torch.tensor([2], dtype=torch.int32, device="cuda") if pool else None
    for t in range(T):
        o = sequence.decay_attention_step(q[:, t], k[:, t], v[:, t], g, S, slots=slots)
    for want in recurrence(k, v, g, torch.zeros(1, H, D, D, device="cuda", dtype=torch.float64)):
        pass
    whole, last = sequence.decay_attention(q, k, v, g)
    bound = 2.0 ** -23 * (1 / g.abs().double()).clamp(max=T).sqrt() + ref.FP32
    for got in (S[-1:], last):
        far = (got.double() - want).flatten(2).norm(dim=2)[0] / want.flatten(2).norm(dim=2)[0]
        assert (far <= bound).all(), (far, bound)
    ref.close(o, torch.matmul(q[:, -1].double().unsqueeze(2), want).squeeze(2) / 4, slack=6)


@pytest.mark.parametrize("n", [1, 3, 64])
def test_short_calls_add_up_to_the_sequence(n):
    """The same in calls of n tokens, the state handed on."""
    from flash_cqt import sequence
    calls, H, D = (6000 if n < 64 else 1500), 5, 16
    gen = torch.Generator().manual_seed(67)
    q, k, v = (randn(gen, 1, calls * n, H, D).cuda() + 0.3 for _ in range(3))
    g = -torch.tensor([0.7, 0.3, 2.0 ** -10.5, 1e-4, 1e-5], device="cuda") / n
    state = torch.zeros(1, H, D, D, device="cuda")
    for t in range(0, calls * n, n):
        _, state = sequence.decay_attention(*(x[:, t:t + n] for x in (q, k, v)), g, state=state)
    left = torch.exp(g.double() * torch.arange(calls * n - 1, -1, -1, device="cuda").unsqueeze(-1))
    want = torch.einsum("th,thi,thj->hij", left, k[0].double(), v[0].double())
    # what each call adds is itself rounded, to FP32 of it, and n additions or fewer come between two decays
    bound = 2.0 ** -23 * (1 / g.abs().double()).clamp(max=calls * n).sqrt() + ref.FP32
    far = (state[0].double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert (far <= bound).all(), (far, bound)


def test_segments_add_up_to_the_sequence():
    """One row of 65600 tokens that the GPU walks in many segments, each carried on by the scan."""
    from flash_cqt import sequence
    T, H, D = 65600, 3, 16
    gen = torch.Generator().manual_seed(71)
    q, k, v = (randn(gen, 1, T, H, D).cuda() + 0.3 for _ in range(3))
    g = -torch.tensor([1e-3, 2e-5, 1.7e-6], device="cuda")
    _, last = sequence.decay_attention(q, k, v, g)
    left = torch.exp(g.double() * torch.arange(T - 1, -1, -1, device="cuda").unsqueeze(-1))
    want = torch.einsum("th,thi,thj->hij", left, k[0].double(), v[0].double())
    far = (last[0].double() - want).flatten(1).norm(dim=1) / want.flatten(1).norm(dim=1)
    assert (far <= 2 * ref.FP32).all(), far
