"""The sequence operators' C entries where the package does not call them."""
import ctypes

import pytest
import torch

import seq_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [(3, 700, 4, 2, 64, 40, True, True), (1, 1500, 2, 2, 128, 128, False, False),
                                  (2, 900, 3, 1, 32, 96, True, False)], ids=str)
def test_gradients_without_the_forward_passes_workspace(case, dtype):
    """starts = NULL: the states that segments start from are made again. The
    gradients are those of a call with them, and of the definition; the
    workspace is used up to its size and not past it."""
    from flash_cqt import _seq_native as n
    lib = n.load()
    B, T, Hq, Hk, Dk, Dv, with_state, ragged = case
    gen = torch.Generator().manual_seed(81)
    q, k, v, go = (torch.randn(B, T, h, d, generator=gen).to(dtype) for h, d in ((Hq, Dk), (Hk, Dk), (Hk, Dv), (Hq, Dv)))
    g, S = -0.3 * torch.rand(Hk, generator=gen), torch.randn(B, Hk, Dk, Dv, generator=gen) if with_state else None
    gl = torch.randn(B, Hk, Dk, Dv, generator=gen)
    lengths = torch.tensor([T * (i + 1) // B - 7 for i in range(B)], dtype=torch.int32) if ragged else None
    kind, stream = n.DTYPES[dtype], n.stream_handle(torch.cuda.current_device())
    at = lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())  # noqa: E731
    dev = [None if t is None else t.cuda() for t in (q, k, v, g, lengths, S, go, gl)]
    Q, K, V, G, L, F, GO, GL = dev

    def room(backward):
        size = lib.fcqt_decay_attention_workspace(B, T, Hq, Hk, Dk, Dv, kind, ragged, backward)
        assert size > 0
        return torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda"), size         # NaN, if it were read
    o, last = torch.empty(B, T, Hq, Dv, dtype=dtype, device="cuda"), torch.empty(B, Hk, Dk, Dv, device="cuda")
    starts, size = room(0)
    n.check(lib.fcqt_decay_attention(n.heads(Q), n.heads(K), n.heads(V), at(G), at(L), at(F), at(last), at(o), at(starts), size,
                                     B, T, Dk, Dv, kind, 0.2, stream), "forward")
    found = []
    for given in (starts, None):
        out = [torch.empty_like(t) for t in (Q, K, V, G)] + [torch.empty(B, Hk, Dk, Dv, device="cuda")]
        work, size = room(2)
        n.check(lib.fcqt_decay_attention_bwd(n.heads(Q), n.heads(K), n.heads(V), at(G), at(L), at(F), at(given), n.heads(GO), at(GL),
                                             *map(at, out), at(work), size, B, T, Dk, Dv, kind, 0.2, stream), "backward")
        torch.cuda.synchronize()
        assert (work[size:] == 255).all()
        found.append(out)
    wide = [None if t is None else t.double().requires_grad_(True) for t in (q, k, v, g, S)]
    wo, wl = ref.decay_attention(*wide[:4], 0.2, wide[4] if with_state else None, lengths)
    want = torch.autograd.grad((wo, wl), [t for t in wide if t is not None], (go.double(), gl.double()))
    for out in found:
        for name, x, y in zip(("dq", "dk", "dv", "dg", "dstate"), out, want):
            if name == "dg":
                assert (x.cpu().double() - y).abs().max() <= 2e-5 * y.abs().max()
            else:
                ref.close(x, y, x.dtype, slack=3.0, what=name)
    # what does not pass through those states is the same, bit for bit
    assert all(torch.equal(found[0][i], found[1][i]) for i in (1, 2, 4))
