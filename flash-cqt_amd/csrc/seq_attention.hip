// Linear attention with a decay for each head, over whole sequences: how its kernels (seq_attention.hpp) are put
// together for a call. A sequence is cut into segments where rows and heads alone are fewer workgroups than the GPU
// wants: each segment's own contribution to the state comes first (k_chunks, states alone), a pass over the segments
// turns them into the states that they start from, and all of them then run at once.
#include <algorithm>

#include "seq_attention.hpp"

using namespace fcqt_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kGrain = 64;          // segments are multiples of this many tokens: whole chunks of every kernel
constexpr int kMaxRows = 65535;     // the grid's last axis

struct Plan {
    int kd, waves, segments;
    int64_t tokens;                 // of a segment
};

int tokens_of_chunk(int32_t dtype) { return chunk_tokens(dtype == FCQT_BF16 ? 1 : 2); }

int padded(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// A kernel with inner dimension kd (padded) and vd columns, 32 a wave, over `tokens` tokens cut into segments of `segment`.
// Two waves where they hold all columns (for 128, twice two would load q and k again: 8 x 7680 bf16 tokens of 8 heads with
// gradients 1446 us, four waves 1023, both with operands of 16 bits).
Plan sized(int kd, int vd, int64_t tokens, int64_t segment) {
    Plan p;
    p.kd = padded(kd);
    p.waves = vd > 64 ? 4 : 2;
    p.tokens = segment;
    p.segments = int((tokens + segment - 1) / segment);
    return p;
}

// [batch][heads][segments][dk][dv] in a workspace; flipped: read with its rows and columns exchanged
State states(float* data, int64_t heads, int64_t segments, int dk, int dv, bool flipped) {
    const int64_t one = int64_t(dk) * dv;
    return {data, heads * segments * one, segments * one, one, flipped ? 1 : dv, flipped ? dv : 1};
}

// The states that segments start from: U[s] (each segment's own) becomes them, in place. back: from the last segment.
// One thread four elements, its segments in turn, loads a few segments ahead.
struct Scan {
    const float* log_decay;
    const int32_t* lengths;
    const float* first;             // [batch][heads][dk][dv] or NULL
    float* last;                    // the states after all of them, or NULL
    float* U;
    int64_t tokens, segment;
    int32_t segments, size, back;
};

__global__ __launch_bounds__(kThreads) void k_scan(Scan a) {
    const int i0 = (blockIdx.x * kThreads + threadIdx.x) * 4;
    if (i0 >= a.size) return;
    const int64_t row = blockIdx.z, at = row * gridDim.y + blockIdx.y;
    const float g = a.log_decay[blockIdx.y];
    const int64_t length = a.lengths ? min(max(int64_t(a.lengths[row]), int64_t(0)), a.tokens) : a.tokens;
    f32x4 x{};
    if (a.first) x = *reinterpret_cast<const f32x4*>(a.first + at * a.size + i0);
    f32x4* U = reinterpret_cast<f32x4*>(a.U + at * a.segments * int64_t(a.size) + i0);
    const int64_t step = a.size / 4;
    // eight segments' loads at a time: one after the other they took 0.5 us each
    for (int j0 = 0; j0 < a.segments; j0 += 8) {
        f32x4 u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = min(j0 + i, a.segments - 1), s = a.back ? a.segments - 1 - j : j;
            u[i] = U[s * step];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = j0 + i, s = a.back ? a.segments - 1 - j : j;
            if (j < a.segments) {
                U[s * step] = x;
                const Decay f(g, int(max(min(a.segment, length - s * a.segment), int64_t(0))));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(f.by, x[e], f.slow ? x[e] : 0.0f) + u[i][e];
            }
        }
    }
    if (a.last) *reinterpret_cast<f32x4*>(a.last + at * a.size + i0) = x;
}

// dg[h] = the sum of one head's slopes: two sets, of `one` and of `two` for each row
__global__ __launch_bounds__(kThreads) void k_slopes(const double* first, const double* second, float* dg, int64_t batch, int one, int two) {
    __shared__ double part[kThreads];
    const int head = blockIdx.x, heads = gridDim.x;
    double sum = 0;
    for (int64_t i = threadIdx.x; i < batch * one; i += kThreads) sum += first[((i / one) * heads + head) * one + i % one];
    for (int64_t i = threadIdx.x; i < batch * two; i += kThreads) sum += second[((i / two) * heads + head) * two + i % two];
    part[threadIdx.x] = sum;
    for (int d = kThreads / 2; d; d /= 2) {
        __syncthreads();
        if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
    }
    if (threadIdx.x == 0) dg[head] = float(part[0]);
}

// Whether every query head of a group has a workgroup of its own: where they share one, its state is updated once, but
// the group's heads are one after the other. 1 x 1958 bf16 tokens, 12 heads on 3, 64 wide: 27 us apart, 48 shared; 8 x 4000,
// 16 heads on 4, 128 wide: 219 apart, 184 shared.
bool spreads(const Plan& p, int64_t batch, int keys, int group) {
    return group > 1 && batch * keys * p.segments < 512;
}

int run(Chunks& a, const Plan& p, bool only_states, int slope, int64_t batch, int heads, int32_t dtype, hipStream_t stream) {
    a.segments = p.segments;
    a.chunks = int32_t(p.tokens / tokens_of_chunk(dtype));
    a.spread = !only_states && !a.reduce && spreads(p, batch, heads, a.group);
    Launch l{p.kd, p.waves, only_states, slope,
             dim3(p.segments, a.spread ? heads * a.group : heads, uint32_t(batch)), stream};
    if (dtype == FCQT_F32) launch_f32(a, l);
    else if (dtype == FCQT_BF16) launch_bf16(a, l);
    else launch_f16(a, l);
    return launched();
}

int scan(const Chunks& a, const float* first, float* last, float* U, int64_t segment, int segments, int size, int64_t batch, int heads,
         hipStream_t stream) {
    Scan s{a.log_decay, a.lengths, first, last, U, a.tokens, segment, segments, size, a.back};
    k_scan<<<dim3((size / 4 + kThreads - 1) / kThreads, heads, uint32_t(batch)), kThreads, 0, stream>>>(s);
    return launched();
}

struct Shape {
    int64_t batch, tokens;
    int hq, hk, dk, dv;
    int32_t dtype;
};

int checked(const fcqt_heads* s, int elem) {
    if (!s || !s->data || s->heads < 1 || s->heads > 65535) return FCQT_EARG;
    // rows are read 16 bytes at a time, and a chunk's with offsets of 32 bits
    if (!aligned(s->data, 16) || ((s->batch_stride | s->token_stride | s->head_stride) * elem) % 16) return FCQT_EALIGN;
    if (s->token_stride < 0 || s->token_stride > (int64_t(1) << 31) / (64 * elem) - FCQT_DECAY_MAX_DIM) return FCQT_EARG;
    return FCQT_OK;
}

int shape_of(Shape& s, int64_t batch, int64_t tokens, int32_t hq, int32_t hk, int32_t dk, int32_t dv, int32_t dtype) {
    if (!known(dtype) || batch < 0 || batch > kMaxRows || tokens < 0 || tokens > (int64_t(1) << 31) - 64) return FCQT_EARG;
    if (hk < 1 || hk > 65535 || hq < hk || hq % hk || hq > 65535) return FCQT_EARG;
    for (int d : {dk, dv})
        if (d < 8 || d > FCQT_DECAY_MAX_DIM || d % 8) return FCQT_EARG;
    s = {batch, tokens, hq, hk, dk, dv, dtype};
    return FCQT_OK;
}

// Tokens of a segment, one cut for the outputs and all gradients. Whole rows are cut into as many workgroups as the GPU
// holds at a time (by the LDS of the main kernels: three on a CU for 16-bit types up to 64 wide, one for fp32 over 64, two
// otherwise). With gradients, 8 x 7680 tokens of 8 heads: 450 us in 768 workgroups, 557 in 512 (bf16, 64 wide), 2349 us in
// 256, 2358 in 512 (fp32, 128 wide); 24 x 4096 tokens of 16 heads, bf16, 64 wide: 1350 us in 768, 1904 in 384. Rows with
// lengths of their own are cut into 1024: half of them ending early leaves half of the workgroups idle (9 rows of 0 to 4097
// tokens: 717 us, 821 with 512). A segment costs a state, written, scanned and read, so none is under 64 tokens
// and the scan's steps stay few beside the chunks that a segment saves: 512 tokens of 64 fp32 heads of 64 take 76 us in
// one segment, 32 in eight.
int64_t segment_of(const Shape& s, bool ragged) {
    const int64_t tokens = std::max<int64_t>(s.tokens, 1);
    const int64_t groups = s.batch * s.hk;
    const bool f32 = s.dtype == FCQT_F32;
    const int64_t held = f32 && s.dk > 64 && s.dv > 64 ? 256 : !f32 && s.dk <= 64 && s.dv <= 64 ? 768 : 512;
    const int64_t fill = ragged ? 1024 : held;
    int64_t want = 1;
    if (4 * groups < 3 * fill && tokens * (s.hq / s.hk) > 256) {
        want = std::max<int64_t>(std::min(fill / groups, tokens / 64), 1);
        while (want > 1 && want * want > 64 * (tokens / 64 + 1)) want = want * 3 / 4;
    }
    const int64_t each = (tokens + want - 1) / want;
    return (each + kGrain - 1) / kGrain * kGrain;
}

int64_t state_floats(const Shape& s, int64_t segment) {
    const int64_t segments = (s.tokens + segment - 1) / segment;
    return segments > 1 ? s.batch * s.hk * segments * s.dk * s.dv : 0;
}

// What the backward pass keeps, in floats: the states that segments start from, both ways (forwards only without those of
// the forward pass); where the decays' gradient
// is wanted, the state's gradient at every chunk's end and the sums.
struct Parts {
    int64_t states, flow, slopes;
    Parts(const Shape& s, const Plan& p, int64_t segment, bool slope) {
        const int64_t groups = s.batch * s.hk * p.waves, chunk = tokens_of_chunk(s.dtype);
        states = state_floats(s, segment);
        flow = slope ? groups * ((s.tokens + chunk - 1) / chunk) * p.kd * 32 : 0;
        slopes = slope ? groups * p.segments : 0;                    // doubles
    }
    int64_t all(int group) const { return 2 * states + flow + 2 * (1 + group) * slopes; }
};

__global__ void k_copy_state(const float* from, float* to, int64_t n) {
    for (int64_t i = (int64_t(blockIdx.x) * kThreads + threadIdx.x) * 4; i < n; i += int64_t(gridDim.x) * kThreads * 4)
        *reinterpret_cast<f32x4*>(to + i) = from ? *reinterpret_cast<const f32x4*>(from + i) : f32x4{};
}

int copy_state(const float* from, float* to, int64_t n, hipStream_t stream) {
    if (!to || !n) return FCQT_OK;
    k_copy_state<<<dim3(uint32_t(std::min<int64_t>((n / 4 + kThreads - 1) / kThreads, 1 << 16))), kThreads, 0, stream>>>(from, to, n);
    return launched();
}

}  // namespace

extern "C" int64_t fcqt_decay_attention_workspace(int64_t batch, int64_t tokens, int32_t hq, int32_t hk, int32_t dk,
                                                  int32_t dv, int32_t dtype, int32_t ragged, int32_t backward) {
    Shape s;
    if (shape_of(s, batch, tokens, hq, hk, dk, dv, dtype) || !batch || !tokens) return 0;
    const int64_t segment = segment_of(s, ragged);
    if (!backward) return state_floats(s, segment) * 4;
    return Parts(s, sized(s.dv, s.dk, s.tokens, segment), segment, backward > 1).all(hq / hk) * 4;
}

extern "C" int fcqt_decay_attention(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v, const float* log_decay,
                                    const int32_t* lengths, const float* state, float* last, void* o, void* workspace,
                                    int64_t workspace_bytes, int64_t batch, int64_t tokens, int32_t dk, int32_t dv,
                                    int32_t dtype, float scale, hipStream_t stream) {
    Shape s;
    if (!q || !k || !v) return FCQT_EARG;
    if (int e = shape_of(s, batch, tokens, q->heads, k->heads, dk, dv, dtype)) return e;
    if (v->heads != k->heads) return FCQT_EARG;
    if (!batch) return FCQT_OK;
    if (!log_decay || !last) return FCQT_EARG;
    if (!aligned(log_decay, 4) || !aligned(lengths, 4) || !aligned(state, 16) || !aligned(last, 16)) return FCQT_EALIGN;
    if (!tokens) return copy_state(state, last, batch * s.hk * dk * dv, stream);
    for (const fcqt_heads* x : {q, k, v})
        if (int e = checked(x, size_of(dtype))) return e;
    if (!o) return FCQT_EARG;
    if (!aligned(o, 16) || !aligned(workspace, 16)) return FCQT_EALIGN;
    if (workspace_bytes < fcqt_decay_attention_workspace(batch, tokens, s.hq, s.hk, dk, dv, dtype, lengths != nullptr, 0)) return FCQT_EARG;
    const int64_t segment = segment_of(s, lengths);
    const Plan p = sized(dk, dv, tokens, segment);
    if (p.segments > 1 && !workspace) return FCQT_EARG;
    float* U = static_cast<float*>(workspace);
    Chunks a{};
    a.q = *q, a.k = *k, a.v = *v, a.log_decay = log_decay, a.lengths = lengths, a.o = o, a.tokens = tokens;
    a.kd = dk, a.vd = dv, a.group = s.hq / s.hk, a.p_scale = scale, a.u_scale = 1, a.x_scale = scale;
    if (p.segments > 1) {
        a.last = states(U, s.hk, p.segments, dk, dv, false);
        if (int e = run(a, p, true, 0, batch, s.hk, dtype, stream)) return e;
        if (int e = scan(a, state, last, U, segment, p.segments, dk * dv, batch, s.hk, stream)) return e;
        a.first = a.last;
        a.last = State{};
    } else {
        a.first = states(const_cast<float*>(state), s.hk, 1, dk, dv, false);
        a.last = states(last, s.hk, 1, dk, dv, false);
    }
    return run(a, p, false, 0, batch, s.hk, dtype, stream);
}

extern "C" int fcqt_decay_attention_bwd(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v,
                                        const float* log_decay, const int32_t* lengths, const float* state,
                                        const void* starts, const fcqt_heads* go, const float* glast, void* dq, void* dk_, void* dv_,
                                        float* dlog_decay, float* dstate, void* workspace, int64_t workspace_bytes,
                                        int64_t batch, int64_t tokens, int32_t dk, int32_t dv, int32_t dtype,
                                        float scale, hipStream_t stream) {
    Shape s;
    if (!q || !k || !v || !go) return FCQT_EARG;
    if (int e = shape_of(s, batch, tokens, q->heads, k->heads, dk, dv, dtype)) return e;
    if (v->heads != k->heads || go->heads != q->heads || !log_decay) return FCQT_EARG;
    if (!aligned(log_decay, 4) || !aligned(lengths, 4) || !aligned(state, 16) || !aligned(starts, 16) ||
        !aligned(glast, 16) || !aligned(dlog_decay, 4) || !aligned(dstate, 16))
        return FCQT_EALIGN;
    const int64_t all = batch * s.hk * dk * dv;
    if (!batch || !tokens) {
        if (dlog_decay) k_slopes<<<dim3(s.hk), kThreads, 0, stream>>>(nullptr, nullptr, dlog_decay, 0, 1, 1);
        if (int e = launched()) return e;
        return copy_state(glast, dstate, all, stream);
    }
    for (const fcqt_heads* x : {q, k, v, go})
        if (int e = checked(x, size_of(dtype))) return e;
    const bool slope = dlog_decay != nullptr;
    const int64_t need = fcqt_decay_attention_workspace(batch, tokens, s.hq, s.hk, dk, dv, dtype, lengths != nullptr, slope ? 2 : 1);
    if (!dq || !dk_ || !dv_ || workspace_bytes < need || (need && !workspace)) return FCQT_EARG;
    if (!aligned(dq, 16) || !aligned(dk_, 16) || !aligned(dv_, 16) || !aligned(workspace, 16)) return FCQT_EALIGN;
    const int64_t segment = segment_of(s, lengths);
    const Plan by_v = sized(dv, dk, tokens, segment), by_k = sized(dk, dv, tokens, segment);
    const Parts part(s, by_v, segment, slope);
    const int segments = by_v.segments;
    float *U = static_cast<float*>(workspace), *R = U + part.states, *flow = R + part.states;
    double* slopes = reinterpret_cast<double*>(flow + part.flow);

    // dv = A(k, q, do) back in time, from the last state's gradient
    Chunks b{};
    b.q = *k, b.k = *q, b.v = *go, b.log_decay = log_decay, b.lengths = lengths, b.tokens = tokens;
    b.kd = dk, b.vd = dv, b.group = s.hq / s.hk, b.back = 1, b.reduce = 1, b.p_scale = scale, b.u_scale = scale, b.x_scale = 1;
    if (segments > 1) {
        b.last = states(R, s.hk, segments, dk, dv, false);
        if (int e = run(b, by_k, true, 0, batch, s.hk, dtype, stream)) return e;
        if (int e = scan(b, glast, dstate, R, segment, segments, dk * dv, batch, s.hk, stream)) return e;
        b.first = b.last;
        b.last = State{};
    } else {
        b.first = states(const_cast<float*>(glast), s.hk, 1, dk, dv, false);
        if (dstate) b.last = states(dstate, s.hk, 1, dk, dv, false);
    }
    b.o = dv_;
    if (int e = run(b, by_k, false, 0, batch, s.hk, dtype, stream)) return e;

    // dk = A(v, do, q) back in time, the same states with rows and columns exchanged
    b.q = *v, b.k = *go, b.v = *q, b.w = *k, b.kd = dv, b.vd = dk, b.o = dk_, b.last = State{};
    b.flow = flow, b.slopes = slopes;
    std::swap(b.first.row, b.first.col);
    if (int e = run(b, by_v, false, slope ? 2 : 0, batch, s.hk, dtype, stream)) return e;

    // dq = A(do, v, k)
    Chunks a{};
    a.q = *go, a.k = *v, a.v = *k, a.w = *q, a.log_decay = log_decay, a.lengths = lengths, a.tokens = tokens;
    a.kd = dv, a.vd = dk, a.group = s.hq / s.hk, a.p_scale = scale, a.u_scale = 1, a.x_scale = scale, a.o = dq;
    if (segments > 1 && starts) {
        a.first = states(const_cast<float*>(static_cast<const float*>(starts)), s.hk, segments, dk, dv, true);
    } else if (segments > 1) {
        a.last = states(U, s.hk, segments, dk, dv, true);
        if (int e = run(a, by_v, true, 0, batch, s.hk, dtype, stream)) return e;
        if (int e = scan(a, state, nullptr, U, segment, segments, dk * dv, batch, s.hk, stream)) return e;
        a.first = a.last;
        a.last = State{};
    } else {
        a.first = states(const_cast<float*>(state), s.hk, 1, dk, dv, true);
    }
    a.flow = flow, a.slopes = slopes + part.slopes;
    if (int e = run(a, by_v, false, slope ? 1 : 0, batch, s.hk, dtype, stream)) return e;
    if (slope) {
        const int per = by_v.segments * by_v.waves;
        k_slopes<<<dim3(s.hk), kThreads, 0, stream>>>(slopes, a.slopes, dlog_decay, batch, per, a.spread ? a.group * per : per);
        return launched();
    }
    return FCQT_OK;
}
