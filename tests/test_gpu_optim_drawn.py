"""8-bit moments over many steps: codes drawn between a value's neighbours
follow AdamW's rule, and are the bits that their definition gives."""
import math

import numpy as np
import pytest
import torch

import seq_ref as ref

HOW = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
F32 = np.float32


# ------------------------------------------------------------ the definition

def mixed(x):
    top = (1 << 64) - 1
    x &= top
    x = (x ^ x >> 32) * 0x9E3779B97F4A7C15 & top
    x = (x ^ x >> 29) * 0xBB67AE8584CAA73B & top
    return x ^ x >> 32


def draws(seed, step, tensor, n):
    """Numbers in [0, 1) for the first and the second moments of a tensor's elements."""
    key = mixed(mixed(seed) + step + (tensor + 1) * 0x9E3779B97F4A7C15)
    x = np.arange(n, dtype=np.uint32) ^ np.uint32(key & 0xFFFFFFFF)
    x = (x ^ x >> np.uint32(16)) * np.uint32(0x9E3779B1) ^ np.uint32(key >> 32)
    x = (x ^ x >> np.uint32(15)) * np.uint32(0xBB67AE85)
    x ^= x >> np.uint32(16)
    return [(y >> np.uint32(8)).astype(F32) * F32(2.0 ** -24) for y in (x * np.uint32(0x9E3779B1), x)]


def encode(x, unsigned, r, least):
    """Codes and scales of x (float32), blocks of 256, by the draws r; least:
    which first moments may become the smallest code."""
    low = 14 if unsigned else 6
    n = len(x)
    a = np.zeros(-(-n // 256) * 256, F32)
    a[:n] = np.abs(x)
    scale = a.reshape(-1, 256).max(1) * F32(1 / 1.9375)
    each = np.repeat(scale, 256)
    y = np.where(each > 0, a / np.where(each > 0, each, F32(1)), F32(0))[:n].astype(F32)
    mags = ref.code_values(unsigned).numpy()[:256 if unsigned else 128]
    c = np.searchsorted(mags, y.astype(np.float64), side="right") - 1               # the code below
    step = np.where(c < 16, 2.0 ** -(low + 4), 2.0 ** (np.maximum(c >> 4, 1) - 5.0 - low))
    f = ((y.astype(np.float64) - mags[c]) / step).astype(F32)                       # exact: 19 bits at most, or y's own
    if unsigned:
        twice = (2 * np.where(c < 16, c, 16 + c % 16)).astype(F32)
        c = c + (r * (twice + F32(1)) < f * (twice + f))
        return np.where(a[:n] > 0, np.clip(c, 1, 255), 0), scale
    c = c + ((r < f) & ((c > 0) | least(scale)))
    return np.minimum(c, 127) | (x < 0).astype(int) << 7, scale


def decode(c, scale, unsigned):
    return ref.code_values(unsigned).numpy()[c].astype(F32) * np.repeat(scale, 256)[:len(c)]


class Plain:
    """One tensor's weights and 8-bit moments, every product and sum rounded on its own."""

    def __init__(self, p):
        n = len(p)
        self.p = p.astype(F32)
        self.m, self.v = (np.zeros(n, np.int64) for _ in range(2))
        self.ms, self.vs = (np.zeros(-(-n // 256), F32) for _ in range(2))

    def step(self, g, seed, step, tensor, lr, betas, eps, weight_decay):
        b1, b2 = betas
        m = decode(self.m, self.ms, False) * F32(b1) + g * F32(1 - b1)
        w = decode(self.v, self.vs, True)
        v = w * w * F32(b2) + g * F32(1 - b2) * g
        w = np.sqrt(v)
        up = m / (w * F32(1 / math.sqrt(1 - b2 ** step)) + F32(eps)) * F32(lr / (1 - b1 ** step))
        self.p = self.p * F32(1 - lr * weight_decay) - up
        rm, rv = draws(seed, step, tensor, len(g))
        each = lambda s: np.repeat(s, 256)[:len(g)]  # noqa: E731
        self.m, self.ms = encode(m, False, rm, lambda s: each(s) * F32(2.0 ** -10) <= w * F32(4))
        self.v, self.vs = encode(w, True, rv, None)


# ----------------------------------------------- of the definition, on the CPU

def test_draws_are_even_and_apart():
    """Means, and products of draws for both moments, of neighbouring elements,
    blocks, steps, tensors and seeds, are those of independent numbers: within
    five of their standard deviations, sqrt(1 / 12 n) and 1 / sqrt(n)."""
    n = 1 << 18
    sets = {(s, t, i): draws(s, t, i, n) for s, t, i in ((0, 1, 0), (0, 2, 0), (0, 1, 1), (1, 1, 0), (0, 1 << 20, 0))}
    base = sets[0, 1, 0]
    for a, b in sets.values():
        for x in (a, b):
            assert abs(x.mean(dtype=np.float64) - 0.5) <= 5 / math.sqrt(12 * n)
            assert abs((x < 2.0 ** -8).mean() - 2.0 ** -8) <= 5 * math.sqrt(2.0 ** -8 / n)
            for lag in (1, 8, 256):
                assert abs(np.corrcoef(x[lag:], x[:-lag])[0, 1]) <= 5 / math.sqrt(n)
        assert abs(np.corrcoef(a, b)[0, 1]) <= 5 / math.sqrt(n)
        if a is not base[0]:
            assert all(abs(np.corrcoef(x, y)[0, 1]) <= 5 / math.sqrt(n) for x in (a, b) for y in base)
    one = np.array([[x[0] for x in draws(3, t, 0, 1)] for t in range(1, 20001)])                # one element, step by step
    assert (abs(one.mean(0) - 0.5) <= 5 / math.sqrt(12 * 20000)).all()
    assert all(abs(np.corrcoef(x[1:], x[:-1])[0, 1]) <= 5 / math.sqrt(20000) for x in one.T)


def test_drawn_codes_keep_the_mean():
    """Over 2000 draws first moments, and the squares of second moments' roots,
    are their values: within five standard deviations of the mean."""
    rng = np.random.default_rng(2)
    x = (rng.standard_normal(256) * np.exp2(-6 * rng.random(256))).astype(F32)
    for unsigned in (False, True):
        values = np.array([decode(*encode(x if not unsigned else abs(x), unsigned, draws(5, t, 0, 256)[unsigned],
                                          lambda s: True), unsigned) for t in range(2000)], np.float64)
        want = x.astype(np.float64)
        if unsigned:
            values, want = values ** 2, want ** 2
        off = abs(values.mean(0) - want)
        assert (off <= 5 * values.std(0) / math.sqrt(2000) + 1e-6 * abs(want)).all()


def test_refusals():
    from flash_cqt import _seq_native as n, optim
    lib, fac = n.load(), n.AdamwFactors(*[0.5] * 8)

    def one(**kw):
        d = dict(p=4096, g=4096, m=4096, v=4096, m_scale=4096, v_scale=4096, n=4)
        d.update(kw)
        return (n.AdamwTensor * 1)(n.AdamwTensor(*d.values()))
    f = lib.fcqt_adamw_drawn
    assert f(None, 0, 0, fac, None, 1, 1, None) == 0 and f(one(n=0), 1, 0, fac, None, 1, 1, None) == 0
    for status, args in ((1, (None, 1, 0, fac)), (1, (one(), 1, 0, None)), (1, (one(), 1, 7, fac)), (1, (one(m_scale=None), 1, 0, fac)),
                         (2, (one(p=4098), 1, 0, fac)), (2, (one(v_scale=4098), 1, 0, fac))):
        assert f(*args, None, 1, 1, None) == status
    assert f(one(), 1, 0, fac, 4098, 1, 1, None) == 2
    for seed in (-1, 1 << 64):
        with pytest.raises(ValueError, match="seed"):
            optim.adamw_step([], [], [], [], step=1, lr=0.1, scales=([], []), seed=seed)
    with pytest.raises(ValueError, match="seed"):
        optim.AdamW([torch.zeros(1)], seed=-1)


# ------------------------------------------------------------------ the kernel

@pytest.mark.gpu
@pytest.mark.parametrize("glue", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_are_the_definitions(dtype, glue, monkeypatch):
    """Weights and codes bit for bit, over steps, in more tensors than one
    launch takes, with blocks of very different sizes and of nothing but zeros."""
    from flash_cqt import _seq_native, optim
    if not glue:
        monkeypatch.setattr(_seq_native, "load_glue", lambda: None)
    rng = np.random.default_rng(3)
    sizes = [1, 7, 255, 256, 257, 2048, 5003] + [11] * 60
    start = [torch.from_numpy(rng.standard_normal(n).astype(F32)).to(dtype) for n in sizes]
    plain = [Plain(p.float().numpy()) for p in start]
    P = [p.cuda() for p in start]
    M, V = ([torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes] for _ in range(2))
    scales = tuple([torch.zeros(-(-n // 256), device="cuda") for n in sizes] for _ in range(2))
    for step in (1, 2, 3, 1000):
        g = [torch.from_numpy((rng.standard_normal(n) * np.exp2(-15 * rng.random(n))).astype(F32)).to(dtype) for n in sizes]
        g[5].zero_()
        g[6][:256] *= 1e-30                                              # a block whose squares vanish
        optim.adamw_step(P, [x.cuda() for x in g], M, V, scales=scales, step=step, seed=12345678901, **HOW)
        for i, (t, x) in enumerate(zip(plain, g)):
            t.step(x.float().numpy(), 12345678901, step, i, **HOW)
            t.p = torch.from_numpy(t.p).to(dtype).float().numpy()
            assert np.array_equal(P[i].float().cpu().numpy(), t.p), (step, i)
            for got, want in ((M[i], t.m), (V[i], t.v), (scales[0][i], t.ms), (scales[1][i], t.vs)):
                assert np.array_equal(got.cpu().numpy(), want), (step, i)


def pair_of_runs(steps, gradient, n, seed=0):
    """An 8-bit and a 32-bit AdamW on the same gradients: (first moments, roots
    of the second) of each, and both weights."""
    from flash_cqt import optim
    ps = [torch.zeros(n, device="cuda", requires_grad=True) for _ in range(2)]
    opts = [optim.AdamW([ps[0]], state_bits=8, seed=seed, **HOW), optim.AdamW([ps[1]], **HOW)]
    gen = torch.Generator("cuda").manual_seed(1)
    for t in range(steps):
        g = gradient(t, torch.randn(n, device="cuda", generator=gen))
        for p, o in zip(ps, opts):
            p.grad = g
            o.step()
    s, w = opts[0].state[ps[0]], opts[1].state[ps[1]]
    (m,), (v,) = optim.read_moments([s["exp_avg"]], [s["exp_avg_sq"]], ([s["exp_avg_scale"]], [s["exp_avg_sq_scale"]]))
    return (m, v.sqrt()), (w["exp_avg"], w["exp_avg_sq"].sqrt()), [p.detach() for p in ps]


@pytest.mark.gpu
def test_8_bit_moments_follow_the_rule():
    """Unit noise, half of every block falling to a tenth after 300 steps and
    another eighth to nothing; 1200 steps later second moments are those of 32
    bits on average. One is drawn between codes 1/16 to 1/32 apart at every
    step and drifts back at (1 - b2) / 2 = 0.5% of itself a step, so its root
    wanders by sqrt(0.045 / 2) = 15% (rms) at most; the mean of 8192 of them by
    0.2%, the mean square by 0.4%. What falls to nothing is left e^-6 of its
    root and no first moment at all."""
    n = 1 << 14
    place = torch.arange(n, device="cuda") % 8
    fallen, gone = (place < 4), place == 4

    def gradient(t, noise):
        return noise if t < 300 else torch.where(fallen, 0.1 * noise, torch.where(gone, torch.zeros_like(noise), noise))
    (m, w), (em, ew), (p, ep) = pair_of_runs(1500, gradient, n)
    for which in (fallen, place > 4):
        ratio = (w[which].square().sum() / ew[which].square().sum()).item()
        assert abs(ratio - 1) <= 0.02, ratio
        assert ((w - ew)[which].norm() / ew[which].norm()).item() <= 0.2
    assert abs((w[gone].mean() / ew[gone].mean()).item() - 1) <= 0.1
    assert not m[gone].any()
    assert ((m - em)[place > 4].norm() / em[place > 4].norm()).item() <= 0.1
    # the weights went the same way: 15% more or less at every step, in either direction
    assert ((p - ep).norm() / ep.norm()).item() <= 0.2


@pytest.mark.gpu
def test_seeds_and_steps():
    """One seed repeats itself; another one, another group and another step draw other codes; resumed runs go on alike."""
    from flash_cqt import optim
    g = torch.randn(8192, device="cuda", generator=torch.Generator("cuda").manual_seed(4))

    def run(seed, steps=3, groups=1):
        ps = [torch.zeros(8192, device="cuda", requires_grad=True) for _ in range(groups)]
        opt = optim.AdamW([dict(params=[p]) for p in ps], state_bits=8, seed=seed)
        for _ in range(steps):
            for p in ps:
                p.grad = g
            opt.step()
        return [opt.state[p]["exp_avg_sq"] for p in ps], opt
    a, b, c = run(0)[0][0], run(0)[0][0], run(1)[0][0]
    assert torch.equal(a, b) and not torch.equal(a, c)
    x, y = run(0, groups=2)[0]
    assert torch.equal(x, a) and not torch.equal(x, y)
    saved = run(9)[1].state_dict()
    q = torch.zeros(8192, device="cuda", requires_grad=True)
    other = optim.AdamW([q], state_bits=8)
    other.load_state_dict(saved)
    assert other.param_groups[0]["seed"] == 9
    del saved["param_groups"][0]["seed"]                                 # one written before there were draws
    other.load_state_dict(saved)
    q.grad = g
    other.step()
