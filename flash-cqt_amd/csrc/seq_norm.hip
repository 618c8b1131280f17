// RMS norm of every head of q and k and their rotation by positions, in one pass, and its gradients.
//
//   n = x rsqrt(mean(x x) + eps),  u = w n,  angle_j = position[axis(j)] freq_j  (one fp32 product)
//   pair (a, b):  (a cos - b sin, a sin + b cos)
//   back:  r = the pairs of dy turned by -angle,  dw = sum n r,  dx = (w r - n mean(n w r)) rsqrt(mean(x x) + eps)
//
// Bound by memory: every element is read once and written once (back: two read, one written). A group of G lanes
// holds a row (one head of one token), V elements a lane in one load of 16 bytes, so the sum of squares and a pair's
// other half stay inside a wave. A workgroup takes whole tokens, whose cosines and sines all their heads share from LDS;
// q's rows first, then k's, two rows' loads under way. Measured: 8 x 7680 fp32 tokens of 8 + 8 heads of 64 in 97 us (5.2
// TB/s; a copy 4.8), 4 x 4099 bf16 tokens of 16 + 4 heads of 128 in 39 us forward (4.3 TB/s) and 63 us back (4.0): there
// a workgroup's start (positions, then sines) is 5% of its time and instructions take over half. Rows of q and k mixed,
// with both weights at hand: 54 and 85 us; one row under way 44 and 74, four 38 and 91 (registers).
#include <algorithm>

#include "seq_common.hpp"

using namespace fcqt_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kTurns = 1024;         // pairs' cosines and sines that a workgroup holds
constexpr int kAhead = 2;           // rows under way
constexpr int kTile = 128;          // most tokens of a tile
constexpr int kBackGroups = 1024;   // most workgroups of the backward pass: rows of partial weight gradients

struct Args {
    fcqt_heads q, k, gq, gk;
    fcqt_rotary rot;
    const float *wq, *wk;
    void *oq, *ok;
    float* partial;
    int64_t tokens, all;            // tokens of a row of the batch, and of all rows
    int32_t dim, pairs, tile;       // tile: tokens that a workgroup takes at a time
    int32_t norm, wide;
    float eps;
};

// Where a tile's tokens lie, in elements: one division a token and not one a row.
struct Places {
    int64_t x[2][kTile], g[2][kTile], pos[kTile];       // of q and k, of their gradients
};

template <bool kBack>
__device__ __forceinline__ void place(const Args& a, int64_t first, int count, Places& at) {
    const int t = threadIdx.x;
    if (t < count) {
        const int64_t token = first + t, row = token / a.tokens, n = token - row * a.tokens;
        at.x[0][t] = row * a.q.batch_stride + n * a.q.token_stride;
        at.x[1][t] = row * a.k.batch_stride + n * a.k.token_stride;
        if (kBack) {
            at.g[0][t] = row * a.gq.batch_stride + n * a.gq.token_stride;
            at.g[1][t] = row * a.gk.batch_stride + n * a.gk.token_stride;
        }
        at.pos[t] = row * a.rot.positions_batch + n * a.rot.axes;
    }
}

// The tile's cosines and sines.
__device__ __forceinline__ void turn(const Args& a, int count, const Places& at, float2 (&cs)[kTurns]) {
    for (int i = threadIdx.x; i < count * a.pairs; i += kThreads) {
        const int t = i / a.pairs, j = i - t * a.pairs;
        int axis = 0;
#pragma unroll
        for (int x = 0; x + 1 < FCQT_ROTARY_AXES; ++x) axis += x + 1 < a.rot.axes && j >= a.rot.ends[x];
        float s, c;
        sincosf(__fmul_rn(a.rot.positions[at.pos[t] + axis], a.rot.freq[j]), &s, &c);
        cs[i] = make_float2(c, s);
    }
}

// The value x of element i turned with its pair's other half; back: by the negative angle.
template <int V, bool kBack>
__device__ __forceinline__ void turned(float (&x)[V], const float2* cs, int at, int pairs, bool interleaved, int lane) {
    if (interleaved) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const int j = (at + e) / 2;
            if (j < pairs) {
                const float c = cs[j].x, s = kBack ? -cs[j].y : cs[j].y;
                const float u = x[e] * c - x[e + 1] * s;
                x[e + 1] = x[e] * s + x[e + 1] * c;
                x[e] = u;
            }
        }
        return;
    }
    const int step = pairs / V;                               // lanes to the other half
    const int other = at < pairs ? lane + step : lane - step;
    const bool mine = at < 2 * pairs;
    const int j = at < pairs ? at : at - pairs;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float y = __shfl(x[e], mine ? other : lane);
        if (mine) {
            const float c = cs[j + e].x, s = kBack ? -cs[j + e].y : cs[j + e].y;
            x[e] = at < pairs ? x[e] * c - y * s : y * s + x[e] * c;
        }
    }
}

template <int G>
__device__ __forceinline__ float group_sum(float x) {
    if (G >= 16) {
        x = sum_of_16(x);
    } else {
#pragma unroll
        for (int d = G / 2; d; d /= 2) x += __shfl_xor(x, d);
    }
    if (G >= 32) x += __shfl_xor(x, 16);
    if (G >= 64) x += __shfl_xor(x, 32);
    return x;
}

// A group's walk over the rows (token of the tile, head) that it takes, step rows apart.
struct Walk {
    int t, h;
    __device__ Walk(int r, int heads) : t(0), h(r) { wrap(heads); }
    __device__ void wrap(int heads) {
        while (h >= heads) h -= heads, ++t;
    }
    __device__ void next(int step, int heads) {
        h += step;
        wrap(heads);
    }
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> raw_row(const void* data, int64_t at, bool wide, bool in) {
    Pack<T, V> y{};
    const T* p = static_cast<const T*>(data) + at;
    if (wide && in) {
        y = *reinterpret_cast<const Pack<T, V>*>(p);
    } else if (in) {
#pragma unroll
        for (int e = 0; e < V; ++e) y.e[e] = p[e];
    }
    return y;
}

template <class T, int V>
__device__ __forceinline__ void widened(const Pack<T, V>& y, float (&x)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = widen<T>(y.e[e]);
}

// q's rows of a tile, then k's: weights, places and sums of one at a time
template <class T, int V, int G>
__global__ __launch_bounds__(kThreads) void k_norm(Args a) {
    __shared__ float2 cs[kTurns];
    __shared__ Places at;
    const int lane = threadIdx.x & 63, col = (threadIdx.x % G) * V, g = threadIdx.x / G;
    constexpr int step = kThreads / G;
    const bool in = col < a.dim;
    const float one = 1.0f / a.dim;
    for (int64_t first = int64_t(blockIdx.x) * a.tile; first < a.all; first += int64_t(gridDim.x) * a.tile) {
        const int count = int(min(int64_t(a.tile), a.all - first));
        __syncthreads();                                       // a tile before this one is done with the places and turns
        place<false>(a, first, count, at);
        __syncthreads();
        for (int key = 0; key < 2; ++key) {
            const fcqt_heads& s = key ? a.k : a.q;
            const float* weights = key ? a.wk : a.wq;
            T* out = static_cast<T*>(key ? a.ok : a.oq) + first * s.heads * a.dim + col;
            auto fetch = [&](const Walk& w) { return raw_row<T, V>(s.data, at.x[key][w.t] + w.h * s.head_stride + col, a.wide, in); };
            // kAhead rows' loads are under way while one is turned
            Walk w(g, s.heads), ahead = w;
            Pack<T, V> held[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (ahead.t < count) held[i] = fetch(ahead);
                ahead.next(step, s.heads);
            }
            float weight[V];
#pragma unroll
            for (int e = 0; e < V; ++e) weight[e] = in && weights ? weights[col + e] : 1.0f;
            if (key == 0 && a.pairs) {
                turn(a, count, at, cs);
                __syncthreads();
            }
            for (int r = g; r < count * s.heads;) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (w.t >= count) break;
                    float x[V];
                    widened<T, V>(held[i], x);
                    if (ahead.t < count) held[i] = fetch(ahead);
                    ahead.next(step, s.heads);
                    if (a.norm) {
                        float sum = 0;
#pragma unroll
                        for (int e = 0; e < V; ++e) sum += x[e] * x[e];
                        const float rstd = rsqrtf(group_sum<G>(sum) * one + a.eps);
#pragma unroll
                        for (int e = 0; e < V; ++e) x[e] = x[e] * rstd * weight[e];
                    }
                    if (a.pairs) turned<V, false>(x, cs + w.t * a.pairs, col, a.pairs, a.rot.interleaved, lane);
                    if (in) store<T, V>(out + int64_t(r) * a.dim, x);
                    w.next(step, s.heads);
                    r += step;
                }
            }
        }
    }
}

template <class T, int V, int G>
__global__ __launch_bounds__(kThreads) void k_norm_bwd(Args a) {
    __shared__ float2 cs[kTurns];
    __shared__ Places at;
    __shared__ float part[kThreads * V];
    const int lane = threadIdx.x & 63, col = (threadIdx.x % G) * V, g = threadIdx.x / G;
    constexpr int step = kThreads / G;
    const bool in = col < a.dim;
    const float one = 1.0f / a.dim;
    for (int key = 0; key < 2; ++key) {
        const fcqt_heads &s = key ? a.k : a.q, &sg = key ? a.gk : a.gq;
        const float* weights = key ? a.wk : a.wq;
        float weight[V], dw[V] = {};
#pragma unroll
        for (int e = 0; e < V; ++e) weight[e] = in && weights ? weights[col + e] : 1.0f;
        for (int64_t first = int64_t(blockIdx.x) * a.tile; first < a.all; first += int64_t(gridDim.x) * a.tile) {
            const int count = int(min(int64_t(a.tile), a.all - first));
            const bool again = key && int64_t(gridDim.x) * a.tile >= a.all;        // a single tile's are there still
            if (!again) {
                __syncthreads();
                place<true>(a, first, count, at);
                __syncthreads();
            }
            T* out = static_cast<T*>(key ? a.ok : a.oq) + first * s.heads * a.dim + col;
            auto fetch = [&](const Walk& w, Pack<T, V>& x, Pack<T, V>& y) {
                x = raw_row<T, V>(s.data, at.x[key][w.t] + w.h * s.head_stride + col, a.wide, in);
                y = raw_row<T, V>(sg.data, at.g[key][w.t] + w.h * sg.head_stride + col, a.wide, in);
            };
            Walk w(g, s.heads), ahead = w;
            Pack<T, V> xs[kAhead], ys[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (ahead.t < count) fetch(ahead, xs[i], ys[i]);
                ahead.next(step, s.heads);
            }
            if (a.pairs && !again) {
                turn(a, count, at, cs);
                __syncthreads();
            }
            for (int r = g; r < count * s.heads;) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (w.t >= count) break;
                    float x[V], y[V];
                    widened<T, V>(xs[i], x);
                    widened<T, V>(ys[i], y);
                    if (ahead.t < count) fetch(ahead, xs[i], ys[i]);
                    ahead.next(step, s.heads);
                    if (a.pairs) turned<V, true>(y, cs + w.t * a.pairs, col, a.pairs, a.rot.interleaved, lane);
                    if (a.norm) {
                        float sum = 0, dot = 0;
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            sum += x[e] * x[e];
                            dot += x[e] * (y[e] * weight[e]);
                        }
                        // n = rstd x: dx = rstd (w r - n mean(n w r))
                        const float rstd = rsqrtf(group_sum<G>(sum) * one + a.eps);
                        const float back = group_sum<G>(dot) * one * rstd * rstd;
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            dw[e] += x[e] * rstd * y[e];
                            y[e] = (y[e] * weight[e] - x[e] * back) * rstd;
                        }
                    }
                    if (in) store<T, V>(out + int64_t(r) * a.dim, y);
                    w.next(step, s.heads);
                    r += step;
                }
            }
        }
        if (!a.partial) continue;
        // the workgroup's groups in a fixed order
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) part[threadIdx.x * V + e] = dw[e];
        __syncthreads();
        for (int d = threadIdx.x; d < a.dim; d += kThreads) {
            float sum = 0;
            for (int j = 0; j < step; ++j) sum += part[j * G * V + d];
            a.partial[(int64_t(blockIdx.x) * 2 + key) * a.dim + d] = sum;
        }
    }
}

// dw[i] = sum over rows of partial[row][i], i < width: eight columns a workgroup, 32 rows at a time (32 columns and
// eight rows took 37 us for 1024 rows: too few loads under way)
__global__ __launch_bounds__(kThreads) void k_norm_dw(const float* partial, float* dw, int rows, int width) {
    __shared__ float part[32][9];
    const int c = threadIdx.x % 8, lane = threadIdx.x / 8, col = blockIdx.x * 8 + c;
    float sum = 0;
    if (col < width) {
#pragma unroll 8
        for (int r = lane; r < rows; r += 32) sum += partial[int64_t(r) * width + col];
    }
    part[lane][c] = sum;
    __syncthreads();
    if (lane == 0 && col < width) {
        for (int r = 1; r < 32; ++r) sum += part[r][c];
        dw[col] = sum;
    }
}

int64_t tile_of(int64_t all, int heads, int pairs, int rows_at_once) {
    // about twelve rows a group (4: 54 us where 12 take 39; 32: 51), but no fewer workgroups than compute units, and the
    // tile's turns in LDS
    int64_t tile = (12 * rows_at_once + heads - 1) / heads;
    tile = std::min<int64_t>({tile, (all + 255) / 256, kTile});
    if (pairs) tile = std::min<int64_t>(tile, kTurns / pairs);
    return std::max<int64_t>(tile, 1);
}

bool placed(const fcqt_heads& s, int bytes, int elem) {
    return aligned(s.data, bytes) && ((s.batch_stride | s.token_stride | s.head_stride) * elem) % bytes == 0;
}

int checked(const fcqt_heads* s, int elem) {
    if (!s || s->heads < 1 || s->heads > 65536 || !s->data) return FCQT_EARG;
    return aligned(s->data, elem) ? FCQT_OK : FCQT_EALIGN;
}

// eight 16-bit or four 32-bit elements a lane: one load of 16 bytes. Halves whose length is no multiple of eight
// lanes' elements turn with four.
int width_of(int32_t dtype, int pairs, bool interleaved) {
    return dtype == FCQT_F32 || (!interleaved && pairs % 8) ? 4 : 8;
}

int group_of(int dim, int v) {
    int g = 4;
    while (g * v < dim) g *= 2;
    return g;
}

int prepare(Args& a, const fcqt_rotary* rot, int64_t batch, int64_t tokens, int32_t dim, int32_t dtype) {
    if (!known(dtype) || batch < 0 || tokens < 0 || dim < 8 || dim > FCQT_SEQ_MAX_DIM || dim % 8) return FCQT_EARG;
    if (tokens && batch > (int64_t(1) << 40) / tokens) return FCQT_EARG;
    a.rot = fcqt_rotary{};
    a.pairs = 0;
    if (rot && rot->axes) {
        if (rot->axes < 0 || rot->axes > FCQT_ROTARY_AXES || !rot->positions || !rot->freq) return FCQT_EARG;
        if (!aligned(rot->positions, 4) || !aligned(rot->freq, 4)) return FCQT_EALIGN;
        a.rot = *rot;
        for (int i = 0, last = 0; i < rot->axes; last = rot->ends[i++])
            if (rot->ends[i] < last) return FCQT_EARG;
        a.pairs = rot->ends[rot->axes - 1];
        if (a.pairs < 0 || 2 * a.pairs > dim || (!rot->interleaved && a.pairs % 4)) return FCQT_EARG;
    }
    a.tokens = tokens;
    a.all = batch * tokens;
    a.dim = dim;
    return FCQT_OK;
}

template <class T, int V, int G>
void launch(const Args& a, bool back, int64_t grid, hipStream_t stream) {
    if (back) k_norm_bwd<T, V, G><<<dim3(uint32_t(grid)), kThreads, 0, stream>>>(a);
    else k_norm<T, V, G><<<dim3(uint32_t(grid)), kThreads, 0, stream>>>(a);
}

template <class T, int V>
void launch(const Args& a, bool back, int64_t grid, hipStream_t stream) {
    switch (group_of(a.dim, V)) {
        case 4: return launch<T, V, 4>(a, back, grid, stream);
        case 8: return launch<T, V, 8>(a, back, grid, stream);
        case 16: return launch<T, V, 16>(a, back, grid, stream);
        case 32: return launch<T, V, 32>(a, back, grid, stream);
        default: return launch<T, V, 64>(a, back, grid, stream);
    }
}

int run(Args& a, bool back, int64_t grid, int32_t dtype, hipStream_t stream) {
    const int v = width_of(dtype, a.pairs, a.rot.interleaved), bytes = v * size_of(dtype);
    a.wide = placed(a.q, bytes, size_of(dtype)) && placed(a.k, bytes, size_of(dtype)) &&
             (!back || (placed(a.gq, bytes, size_of(dtype)) && placed(a.gk, bytes, size_of(dtype))));
    if (!aligned(a.oq, bytes) || !aligned(a.ok, bytes)) return FCQT_EALIGN;
    if (dtype == FCQT_F32) launch<float, 4>(a, back, grid, stream);
    else if (dtype == FCQT_BF16 && v == 8) launch<bf16, 8>(a, back, grid, stream);
    else if (dtype == FCQT_BF16) launch<bf16, 4>(a, back, grid, stream);
    else if (v == 8) launch<f16, 8>(a, back, grid, stream);
    else launch<f16, 4>(a, back, grid, stream);
    return launched();
}

int64_t back_groups(const Args& a) { return std::min<int64_t>(kBackGroups, (a.all + a.tile - 1) / a.tile); }

}  // namespace

extern "C" int fcqt_head_norm_rotary(const fcqt_heads* q, const fcqt_heads* k, const fcqt_rotary* rot, const float* wq,
                                     const float* wk, void* q_out, void* k_out, int64_t batch, int64_t tokens,
                                     int32_t dim, int32_t dtype, int32_t norm, float eps, hipStream_t stream) {
    Args a{};
    if (int e = prepare(a, rot, batch, tokens, dim, dtype)) return e;
    if (a.all == 0) return FCQT_OK;
    if (int e = checked(q, size_of(dtype))) return e;
    if (int e = checked(k, size_of(dtype))) return e;
    if (!q_out || !k_out) return FCQT_EARG;
    if (!aligned(wq, 4) || !aligned(wk, 4)) return FCQT_EALIGN;
    a.q = *q, a.k = *k, a.wq = wq, a.wk = wk, a.oq = q_out, a.ok = k_out, a.norm = norm, a.eps = eps;
    const int v = width_of(dtype, a.pairs, a.rot.interleaved);
    a.tile = int32_t(tile_of(a.all, q->heads + k->heads, a.pairs, kThreads / group_of(dim, v)));
    const int64_t grid = std::min<int64_t>((a.all + a.tile - 1) / a.tile, 1 << 22);
    return run(a, false, grid, dtype, stream);
}

// (the same for all shapes but the head dimension)
extern "C" int64_t fcqt_head_norm_rotary_partial(int64_t, int64_t, int32_t, int32_t dim, int32_t) {
    return int64_t(kBackGroups) * 2 * dim;
}

extern "C" int fcqt_head_norm_rotary_bwd(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* gq,
                                         const fcqt_heads* gk, const fcqt_rotary* rot, const float* wq, const float* wk,
                                         void* dq, void* dk, float* dw, float* partial, int64_t batch, int64_t tokens,
                                         int32_t dim, int32_t dtype, int32_t norm, float eps, hipStream_t stream) {
    Args a{};
    if (int e = prepare(a, rot, batch, tokens, dim, dtype)) return e;
    if (!dw != !partial) return FCQT_EARG;
    if (!aligned(wq, 4) || !aligned(wk, 4) || !aligned(dw, 4) || !aligned(partial, 4)) return FCQT_EALIGN;
    int64_t grid = 0;
    if (a.all) {
        for (const fcqt_heads* s : {q, k, gq, gk})
            if (int e = checked(s, size_of(dtype))) return e;
        if (!dq || !dk || q->heads != gq->heads || k->heads != gk->heads) return FCQT_EARG;
        a.q = *q, a.k = *k, a.gq = *gq, a.gk = *gk, a.wq = wq, a.wk = wk, a.oq = dq, a.ok = dk, a.norm = norm, a.eps = eps;
        a.partial = partial;
        const int v = width_of(dtype, a.pairs, a.rot.interleaved);
        a.tile = int32_t(tile_of(a.all, q->heads + k->heads, a.pairs, kThreads / group_of(dim, v)));
        grid = back_groups(a);
        if (int e = run(a, true, grid, dtype, stream)) return e;
    }
    if (!dw) return FCQT_OK;
    k_norm_dw<<<dim3((2 * dim + 7) / 8), kThreads, 0, stream>>>(partial, dw, int(grid), 2 * dim);
    return launched();
}
