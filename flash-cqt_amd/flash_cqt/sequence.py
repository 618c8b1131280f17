"""Operators of a sequence model over CQT frames, on hand-written HIP kernels
(libflashcqt_seq.so): what a program trains on whole signals and runs one hop
at a time beside TrainableCQT and SlicedCQT.

    q, k = head_norm_rotary(q, k, positions, freq, sections, wq, wk)
    o, state = decay_attention(q, k, v, log_decay, state=state, lengths=lengths)
    o = decay_attention_step(q, k, v, log_decay, states, slots=slots)

Tensors are float32, bfloat16 or float16 on one GPU; sums, norms and states
are float32. head_norm_rotary and decay_attention record gradients (tangents
of forward mode raise). Work goes
to the current stream of the tensors' device, which must be the current one.
Strided inputs are read in place where their last dimension is contiguous.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _seq_native as _n

__all__ = ["rotary_frequencies", "head_norm_rotary", "decay_attention", "decay_attention_step"]


def _glue():
    """The host glue where it may stand in for the Python paths, else None."""
    return None if torch.compiler.is_compiling() else _n.load_glue()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


_ORDINARY = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def _plain(*tensors):
    return _ORDINARY.issuperset(map(type, tensors))


def _in_place(t):
    """t, or a contiguous copy where the kernels cannot read it as it lies."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _heads_of(name, t, dims, dtype=None, device=None):
    _need(torch.is_tensor(t) and t.dim() == dims, f"{name} must be a tensor of {dims} dimensions")
    _need(t.is_cuda, f"{name} is on {t.device}: the operator needs a GPU")
    _need(t.dtype in _n.DTYPES, f"{name} is {t.dtype}: float32, bfloat16 or float16 wanted")
    _need(dtype is None or t.dtype == dtype, f"{name} is {t.dtype}, q is {dtype}")
    _need(device is None or t.device == device, f"{name} is on {t.device}, q on {device}")
    d = t.shape[-1]
    _need(8 <= d <= _n.MAX_DIM and d % 8 == 0, f"{name} has heads of {d}: a multiple of 8 up to {_n.MAX_DIM} wanted")
    _need(t.shape[-2] >= 1, f"{name} has no heads")


def _floats(name, t, shape, device):
    """t as contiguous float32 of the shape, on the device."""
    _need(torch.is_tensor(t) and tuple(t.shape) == tuple(shape), f"{name} must have the shape {tuple(shape)}")
    _need(t.dtype == torch.float32, f"{name} is {t.dtype}: float32 wanted")
    _need(t.device == device, f"{name} is on {t.device}, q on {device}")
    return t.contiguous()


def _aligned(t):
    """t, contiguous, or a copy at a multiple of 16 bytes."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _keep(ctx, *tensors):
    """Save tensors for the backward pass, and what they are."""
    ctx.kept = [None if t is None else (t.shape, t.dtype, t.device) for t in tensors]
    ctx.save_for_backward(*tensors)


def _kept(ctx):
    """The saved tensors, as saved-tensor hooks may have changed them: of any strides, but nothing else."""
    tensors = ctx.saved_tensors
    if any(k is not None and k != (t.shape, t.dtype, t.device) for k, t in zip(ctx.kept, tensors)):
        raise RuntimeError("a saved tensor came back with another shape, type or device")
    return tensors


def _contiguous(*tensors):
    return [None if t is None else t.contiguous() for t in tensors]


# ------------------------------------------------- head norm and rotary positions

def rotary_frequencies(sections, base=10000.0, device="cuda"):
    """Angles of one position for each pair: base ** (-j / n) for the j-th of
    an axis's n pairs. sections: pairs of each axis; base: one, or one for each
    axis."""
    bases = [base] * len(sections) if isinstance(base, (int, float)) else list(base)
    _need(len(bases) == len(sections), "one base, or one for each axis")
    return torch.cat([float(b) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
                      for n, b in zip(sections, bases)]).float().to(device)


def head_norm_rotary(q, k, positions=None, freq=None, sections=(), wq=None, wk=None, *, eps=1e-6, interleaved=False,
                     norm=True):
    """RMS norm of every head of q and k, times wq and wk, then the rotation by
    positions on one to four axes (frame, octave, bin of the octave, ...), in
    one pass; returns the new (q, k), contiguous.

    q [B, T, Hq, D], k [B, T, Hk, D]. wq, wk: float32 [D], or None (ones).
    positions: [T, A] or [B, T, A], float32 (fractional ones among them) or
    whole numbers; freq: float32 [sum(sections)] (rotary_frequencies), the
    angle of each pair for a position of one; sections: how many pairs each of
    the A axes turns, in order. The angle is the float32 product of the two.
    Pairs are (j, j + sum(sections)) or, interleaved, (2j, 2j + 1); elements
    past the last pair stay. positions=None: no rotation; norm=False: rotation
    alone. Gradients go to q, k, wq and wk; positions and freq are needed for
    them, so neither may be changed in place before the backward pass."""
    glue = _glue()
    if glue is not None and _plain(q, k, positions, freq, wq, wk):
        out = glue.norm_rotary(q, k, positions, freq, sections, wq, wk, eps, interleaved, norm)
        if out is not None:
            return out
    _n.no_tangents(q, k, positions, freq, wq, wk)
    _heads_of("q", q, 4)
    _heads_of("k", k, 4, q.dtype, q.device)
    B, T, _, D = q.shape
    _need(k.shape[0] == B and k.shape[1] == T and k.shape[3] == D,
          f"k {tuple(k.shape)} and q {tuple(q.shape)} differ in more than their heads")
    _need(norm or (wq is None and wk is None), "weights belong to the norm")
    _need(eps >= 0, "eps must not be negative")
    wq, wk = (w if w is None else _floats(n, w, (D,), q.device) for n, w in (("wq", wq), ("wk", wk)))
    sections = tuple(int(n) for n in sections)
    if positions is None:
        _need(not sections and freq is None, "freq and sections without positions")
    else:
        A, pairs = len(sections), sum(sections)
        _need(1 <= A <= _n.ROTARY_AXES, f"{A} axes: 1 to {_n.ROTARY_AXES} wanted")
        _need(min(sections) >= 0 and 2 * pairs <= D, f"sections {sections} do not fit heads of {D}")
        _need(interleaved or pairs % 4 == 0, f"{pairs} pairs: a multiple of 4 wanted unless interleaved")
        _need(torch.is_tensor(positions) and tuple(positions.shape) in ((T, A), (B, T, A)),
              f"positions must have the shape {(T, A)} or {(B, T, A)}")
        _need(positions.device == q.device, f"positions are on {positions.device}, q on {q.device}")
        positions = positions.detach().float().contiguous()
        _need(freq is not None, "positions without freq")
        freq = _floats("freq", freq.detach(), (pairs,), q.device)
    how = (sections, float(eps), bool(interleaved), bool(norm))
    if _wants_grad(q, k, wq, wk):
        return _HeadNormRotary.apply(q, k, wq, wk, _saved(positions), _saved(freq), how)
    return _head_norm_rotary(q, k, wq, wk, positions, freq, how)


def _saved(t):
    """t as it can be saved for the backward pass."""
    return t.clone() if t is not None and t.is_inference() else t


def _rotary(positions, freq, how):
    sections, _, interleaved, _ = how
    r = _n.Rotary()
    if positions is not None and sum(sections):
        r.positions, r.freq = positions.data_ptr(), freq.data_ptr()
        r.positions_batch = positions[0].numel() if positions.dim() == 3 else 0
        r.axes, r.interleaved = len(sections), interleaved
        end = 0
        for i, n in enumerate(sections):
            end += n
            r.ends[i] = end
    return r


def _ptr(t):
    return None if t is None else t.data_ptr()


def _head_norm_rotary(q, k, wq, wk, positions, freq, how):
    q, k = _in_place(q), _in_place(k)
    B, T, _, D = q.shape
    oq, ok = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    if B * T:
        _n.check(_n.load().fcqt_head_norm_rotary(_n.heads(q), _n.heads(k), _rotary(positions, freq, how), _ptr(wq),
                                                 _ptr(wk), oq.data_ptr(), ok.data_ptr(), B, T, D, _n.DTYPES[q.dtype],
                                                 how[3], how[1], _n.stream_handle(q.device.index)), "head_norm_rotary")
    return oq, ok


class _HeadNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, freq, how):
        ctx.how = how
        _keep(ctx, q, k, wq, wk, positions, freq)
        return _head_norm_rotary(q, k, wq, wk, positions, freq, how)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, positions, freq = _kept(ctx)
        wq, wk, positions, freq = _contiguous(wq, wk, positions, freq)
        how = ctx.how
        q, k, gq, gk = (_in_place(t) for t in (q, k, gq, gk))
        B, T, _, D = q.shape
        dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        dw = None
        if wq is not None or wk is not None:
            dw = torch.zeros(2, D, dtype=torch.float32, device=q.device) if B * T == 0 else \
                torch.empty(2, D, dtype=torch.float32, device=q.device)
        if B * T:
            lib = _n.load()
            kind = _n.DTYPES[q.dtype]
            partial = dw if dw is None else torch.empty(
                lib.fcqt_head_norm_rotary_partial(B, T, q.shape[2] + k.shape[2], D, kind), dtype=torch.float32, device=q.device)
            _n.check(lib.fcqt_head_norm_rotary_bwd(_n.heads(q), _n.heads(k), _n.heads(gq), _n.heads(gk),
                                                   _rotary(positions, freq, how), _ptr(wq), _ptr(wk), dq.data_ptr(),
                                                   dk.data_ptr(), _ptr(dw), _ptr(partial), B, T, D, kind, how[3], how[1],
                                                   _n.stream_handle(q.device.index)), "head_norm_rotary backward")
        return dq, dk, None if wq is None else dw[0], None if wk is None else dw[1], None, None, None


# ------------------------------------------------------- attention with a decay

def _attention_inputs(q, k, v, log_decay, dims, lead):
    _heads_of("q", q, dims)
    _heads_of("k", k, dims, q.dtype, q.device)
    _heads_of("v", v, dims, q.dtype, q.device)
    _need(k.shape[:lead] == q.shape[:lead] and v.shape[:lead] == q.shape[:lead] and k.shape[-1] == q.shape[-1]
          and v.shape[-2] == k.shape[-2], f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    _need(q.shape[-2] % k.shape[-2] == 0, f"{q.shape[-2]} query heads cannot share {k.shape[-2]} key heads")
    return _floats("log_decay", log_decay, (k.shape[-2],), q.device)


def decay_attention(q, k, v, log_decay, *, scale=None, state=None, lengths=None):
    """Linear attention with a decay for each head, over whole sequences:
    S_t = exp(log_decay) S_{t-1} + k_t v_t^T, o_t = scale q_t S_t; returns
    (o [B, T, Hq, Dv], the last states [B, Hk, Dk, Dv]).

    q [B, T, Hq, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv]; Hq is a multiple of
    Hk, and Hq / Hk neighbouring query heads share a key head. log_decay:
    float32 [Hk], zero or below (-inf forgets at once); scale: Dk ** -0.5
    unless given. state: float32 [B, Hk, Dk, Dv], the states before the first
    token (None: zero), what an earlier call returned. lengths: int32 [B],
    valid tokens of each row (None: all); what lies past them may be anything,
    o is zero there and the last state is the one at the length. Gradients go
    to q, k, v, log_decay and state. Dk and Dv are at most 128. The sequence
    is computed in chunks of up to 64 tokens: a value that is not finite, or
    over bfloat16's largest (3.38e38), makes NaN, in the tokens before it in
    its chunk too."""
    glue = _glue()
    if glue is not None and _plain(q, k, v, log_decay, state, lengths):
        out = glue.attention(q, k, v, log_decay, state, lengths, scale)
        if out is not None:
            return out
    _n.no_tangents(q, k, v, log_decay, state)
    decay = _attention_inputs(q, k, v, log_decay, 4, 2)
    B, T, Hq, Dk = q.shape
    Hk, Dv = v.shape[2:]
    _need(max(Dk, Dv) <= _n.DECAY_MAX_DIM, f"heads of {Dk} and {Dv}: at most {_n.DECAY_MAX_DIM}")
    _need(B <= 65535, f"{B} rows: at most 65535 in one call")
    if state is not None:
        state = _aligned(_floats("state", state, (B, Hk, Dk, Dv), q.device))
    if lengths is not None:
        _need(torch.is_tensor(lengths) and lengths.dtype == torch.int32 and tuple(lengths.shape) == (B,)
              and lengths.device == q.device, f"lengths must be an int32 tensor [{B}] beside q")
        lengths = lengths.contiguous()
    scale = Dk ** -0.5 if scale is None else float(scale)
    if _wants_grad(q, k, v, decay, state):
        return _DecayAttention.apply(q, k, v, decay, state, lengths, scale)
    return _decay_attention(q, k, v, decay, state, lengths, scale)[:2]


def _wide(t):
    """t, or a contiguous copy where the kernels cannot read it 16 bytes at a
    time (or its tokens lie too far apart for their 32-bit offsets)."""
    e = t.element_size()
    b, n, h, d = t.stride()
    ok = (d == 1 and t.data_ptr() % 16 == 0 and (b | n | h) * e % 16 == 0
          and 0 <= n <= (1 << 31) // (64 * e) - _n.DECAY_MAX_DIM)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _workspace(q, k, v, lengths, backward):
    B, T, Hq, Dk = q.shape
    n = _n.load().fcqt_decay_attention_workspace(B, T, Hq, k.shape[2], Dk, v.shape[3], _n.DTYPES[q.dtype],
                                                 lengths is not None, backward)
    return torch.empty(n, dtype=torch.uint8, device=q.device), n


def _decay_attention(q, k, v, decay, state, lengths, scale):
    q, k, v = _wide(q), _wide(k), _wide(v)
    B, T, Hq, Dk = q.shape
    Hk, Dv = v.shape[2:]
    o = torch.empty(B, T, Hq, Dv, dtype=q.dtype, device=q.device)
    last = torch.empty(B, Hk, Dk, Dv, dtype=torch.float32, device=q.device)
    work, size = _workspace(q, k, v, lengths, 0)
    _n.check(_n.load().fcqt_decay_attention(
        _n.heads(q), _n.heads(k), _n.heads(v), decay.data_ptr(), _ptr(lengths), _ptr(state), last.data_ptr(),
        o.data_ptr(), work.data_ptr(), size, B, T, Dk, Dv, _n.DTYPES[q.dtype], scale,
        _n.stream_handle(q.device.index)), "decay_attention")
    return o, last, work


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        o, last, work = _decay_attention(q, k, v, decay, state, lengths, scale)
        _keep(ctx, q, k, v, decay, state, lengths, work)                # work: the states that segments start from
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, go, glast):
        if go is None and glast is None:
            return (None,) * 7
        q, k, v, decay, state, lengths, starts = _kept(ctx)
        decay, state, lengths, starts = _contiguous(decay, state, lengths, starts)
        state, starts = _aligned(state), _aligned(starts)
        B, T, Hq, Dk = q.shape
        Hk, Dv = v.shape[2:]
        go = torch.zeros(B, T, Hq, Dv, dtype=q.dtype, device=q.device) if go is None else _wide(go)
        glast = None if glast is None else _aligned(glast.contiguous())
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dg = torch.empty_like(decay) if ctx.needs_input_grad[3] else None
        ds = torch.empty_like(state) if state is not None and ctx.needs_input_grad[4] else None
        q, k, v = _wide(q), _wide(k), _wide(v)
        work, size = _workspace(q, k, v, lengths, 1 if dg is None else 2)
        _n.check(_n.load().fcqt_decay_attention_bwd(
            _n.heads(q), _n.heads(k), _n.heads(v), decay.data_ptr(), _ptr(lengths), _ptr(state),
            starts.data_ptr() or None, _n.heads(go), _ptr(glast), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(dg), _ptr(ds), work.data_ptr(), size, B, T,
            Dk, Dv, _n.DTYPES[q.dtype], ctx.scale, _n.stream_handle(q.device.index)), "decay_attention backward")
        return dq, dk, dv, dg, ds, None, None


def decay_attention_step(q, k, v, log_decay, state, *, slots=None, scale=None):
    """One token of every running sequence: S <- exp(log_decay) S + k v^T, in
    place, and o = scale q S; returns o [B, Hq, Dv].

    q [B, Hq, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; Hq is a multiple of Hk, and
    Hq / Hk neighbouring query heads share a key head. log_decay: float32
    [Hk], zero or below; scale: Dk ** -0.5 unless given. state: float32
    [pool, Hk, Dk, Dv], contiguous, at a multiple of 16 bytes. slots: int32
    [B], the state of each row,
    without repeats, or None: row b has state b. A row whose slot is outside
    the pool (-1, say) has no sequence: its o is zero and no state changes.
    No gradients: decay_attention records them, over whole sequences."""
    glue = _glue()
    if glue is not None and _plain(q, k, v, log_decay, state, slots):
        out = glue.step(q, k, v, log_decay, state, slots, scale)
        if out is not None:
            return out
    _n.no_tangents(q, k, v, log_decay, state)
    decay = _attention_inputs(q, k, v, log_decay, 3, 1)
    _need(not _wants_grad(q, k, v, log_decay, state), "decay_attention_step records no gradients: use decay_attention")
    B, Hq, Dk = q.shape
    Hk, Dv = v.shape[1:]
    _need(torch.is_tensor(state) and state.dtype == torch.float32 and state.device == q.device
          and state.dim() == 4 and tuple(state.shape[1:]) == (Hk, Dk, Dv) and state.is_contiguous(),
          f"state must be a contiguous float32 tensor [pool, {Hk}, {Dk}, {Dv}] beside q")
    if slots is None:
        _need(state.shape[0] >= B, f"{state.shape[0]} states for {B} rows")
    else:
        _need(torch.is_tensor(slots) and slots.dtype == torch.int32 and tuple(slots.shape) == (B,)
              and slots.device == q.device, f"slots must be an int32 tensor [{B}] beside q")
        slots = slots.contiguous()
    q, k, v = (_in_place(t).unsqueeze(1) for t in (q, k, v))
    o = torch.empty(B, Hq, Dv, dtype=q.dtype, device=q.device)
    if B:
        _n.check(_n.load().fcqt_decay_attention_step(
            _n.heads(q), _n.heads(k), _n.heads(v), decay.data_ptr(), state.data_ptr(), _ptr(slots), o.data_ptr(), B,
            state.shape[0], Dk, Dv, _n.DTYPES[q.dtype], Dk ** -0.5 if scale is None else float(scale),
            _n.stream_handle(q.device.index)), "decay_attention_step")
        torch.autograd.graph.increment_version([state])
    return o
