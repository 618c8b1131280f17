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
