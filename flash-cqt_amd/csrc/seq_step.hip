// Linear attention with a decay for each head, one token of every running sequence:
//
//   S <- exp(g) S + k v',   o = scale q S
//
// exp(g) S is S + expm1(g) S in one rounding where g > -1/2: exp(g) itself, rounded near one, would be off by the same
// 2^-25 and more at every token, which adds up over a head's horizon (g = -1e-4: 2e-4 of the state after 60000 tokens, so
// 3e-6).
//
// Bound by memory: the states, dk x dv fp32 a head, are read and written once; everything else is small. A workgroup
// takes a slice of the columns of one head's state, four columns a thread, rows spread over the rest: the slice stays
// in registers between its load, its store and the products with every query head of the group. 255 sequences' 16 heads of
// 128 x 128 take 112 us with states that come from HBM (4.8 TB/s, as a copy), 78 us where the 268 MB stay in the memory-side
// cache from call to call; one sequence's 3 us, of 6 us with its host part.
#include <algorithm>

#include "seq_common.hpp"

using namespace fcqt_seq;

namespace {

constexpr int kThreads = 256;

struct Args {
    fcqt_heads q, k, v;
    const float* log_decay;
    float* state;
    const int32_t* slots;
    void* o;
    int64_t pool;
    int32_t dk, dv;
    float scale;
};

template <class T>
__device__ __forceinline__ float element(const fcqt_heads& s, int64_t row, int head, int i) {
    return widen<T>(static_cast<const T*>(s.data)[row * s.batch_stride + head * s.head_stride + i]);
}

// kCols: threads along the columns, of four each; kRows: rows of the state that a thread holds at most
template <class T, int kCols, int kRows>
__global__ __launch_bounds__(kThreads) void k_step(Args a) {
    constexpr int kLanes = kThreads / kCols;               // threads along the rows
    __shared__ float qs[FCQT_SEQ_MAX_DIM], ks[FCQT_SEQ_MAX_DIM];
    __shared__ float part[4][kCols * 4];
    const int64_t row = blockIdx.z;
    const int head = blockIdx.y, group = a.q.heads / a.k.heads;
    const int cl = threadIdx.x % kCols, rl = threadIdx.x / kCols, col = (blockIdx.x * kCols + cl) * 4;
    const bool in = col < a.dv;
    const int64_t slot = a.slots ? a.slots[row] : row;
    T* o = static_cast<T*>(a.o) + (row * a.q.heads + int64_t(head) * group) * a.dv;
    if (slot < 0 || slot >= a.pool) {
        for (int i = threadIdx.x; i < group * kCols * 4; i += kThreads) {
            const int c = blockIdx.x * kCols * 4 + i % (kCols * 4);
            if (c < a.dv) o[int64_t(i / (kCols * 4)) * a.dv + c] = narrow<T>(0.0f);
        }
        return;
    }
    float* s = a.state + ((slot * a.k.heads + head) * a.dk) * int64_t(a.dv) + col;
    float x[kRows][4];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = rl + i * kLanes;
        if (in && r < a.dk) load<float, 4>(s + int64_t(r) * a.dv, x[i]);
    }
    for (int i = threadIdx.x; i < a.dk; i += kThreads) ks[i] = element<T>(a.k, row, head, i);
    float v[4] = {};
    if (in) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = element<T>(a.v, row, head, col + e);
    }
    const float g = a.log_decay[head];
    const bool slow = g > -0.5f;
    const float decay = slow ? expm1f(g) : expf(g);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = rl + i * kLanes;
        if (in && r < a.dk) {
            const float kr = ks[r];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = fmaf(decay, x[i][e], slow ? x[i][e] : 0.0f) + kr * v[e];
            store<float, 4>(s + int64_t(r) * a.dv, x[i]);
        }
    }
    for (int h = 0; h < group; ++h) {
        __syncthreads();
        for (int i = threadIdx.x; i < a.dk; i += kThreads) qs[i] = element<T>(a.q, row, head * group + h, i);
        __syncthreads();
        float sum[4] = {};
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = rl + i * kLanes;
            if (in && r < a.dk) {
                const float qr = qs[r];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += qr * x[i][e];
            }
        }
        // the wave's row lanes, then the four waves in order
#pragma unroll
        for (int d = 32; d >= kCols; d /= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], d);
        if (threadIdx.x % 64 < kCols) {
#pragma unroll
            for (int e = 0; e < 4; ++e) part[threadIdx.x / 64][cl * 4 + e] = sum[e];
        }
        __syncthreads();
        if (threadIdx.x < kCols * 4) {
            const int c = blockIdx.x * kCols * 4 + threadIdx.x;
            if (c < a.dv) {
                float y = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) y += part[w][threadIdx.x];
                o[int64_t(h) * a.dv + c] = narrow<T>(y * a.scale);
            }
        }
    }
}

template <class T, int kCols>
void launch(const Args& a, dim3 grid, hipStream_t stream) {
    const int rows = (a.dk + kThreads / kCols - 1) / (kThreads / kCols);
    if (rows <= 2) k_step<T, kCols, 2><<<grid, kThreads, 0, stream>>>(a);
    else if (rows <= 4) k_step<T, kCols, 4><<<grid, kThreads, 0, stream>>>(a);
    else if (rows <= 8) k_step<T, kCols, 8><<<grid, kThreads, 0, stream>>>(a);
    else if (rows <= 16) k_step<T, kCols, 16><<<grid, kThreads, 0, stream>>>(a);
    else k_step<T, kCols, 32><<<grid, kThreads, 0, stream>>>(a);
}

template <class T>
void launch(const Args& a, int64_t batch, hipStream_t stream) {
    // Slices of 64 columns, or of 32 where that is fewer than two workgroups on a compute unit (7 x 16 heads of 128 x 128
    // take 4.6 us so, 7.1 in slices of 128; 40 x 16: 15.4 against 14.3 in slices of 64; 64 of 128 x 16: 20.6, slices of 128
    // 21.5; 90 x 8 heads of 256 x 64: 15.0, 32 columns 15.9, 128 columns 26.0), or of 128 where a row is no whole
    // number of slices, whose rims two workgroups would share (200 x 16 heads of 96 x 80: 33.6 us, 43.1 in slices of 64).
    const auto grid = [&](int columns) { return dim3((a.dv + columns - 1) / columns, a.k.heads, uint32_t(batch)); };
    if (batch * a.k.heads * ((a.dv + 63) / 64) < 512) launch<T, 8>(a, grid(32), stream);
    else if (a.dv < 64 || a.dv % 64 == 0) launch<T, 16>(a, grid(64), stream);
    else launch<T, 32>(a, grid(128), stream);
}

}  // namespace

extern "C" int fcqt_decay_attention_step(const fcqt_heads* q, const fcqt_heads* k, const fcqt_heads* v,
                                         const float* log_decay, float* state, const int32_t* slots, void* o,
                                         int64_t batch, int64_t pool, int32_t dk, int32_t dv, int32_t dtype,
                                         float scale, hipStream_t stream) {
    if (!known(dtype) || batch < 0 || pool < 0 || dk < 8 || dv < 8 || dk % 8 || dv % 8 || dk > FCQT_SEQ_MAX_DIM ||
        dv > FCQT_SEQ_MAX_DIM)
        return FCQT_EARG;
    if (batch == 0) return FCQT_OK;
    if (!q || !k || !v || !q->data || !k->data || !v->data || !log_decay || !o || (pool && !state)) return FCQT_EARG;
    if (k->heads < 1 || k->heads > 65535 || v->heads != k->heads || q->heads < k->heads || q->heads % k->heads) return FCQT_EARG;
    if (!slots && batch > pool) return FCQT_EARG;
    const int elem = size_of(dtype);
    if (!aligned(q->data, elem) || !aligned(k->data, elem) || !aligned(v->data, elem) || !aligned(o, elem) ||
        !aligned(log_decay, 4) || !aligned(slots, 4) || !aligned(state, 16))
        return FCQT_EALIGN;
    // the grid's last axis holds 65535 rows
    for (int64_t at = 0; at < batch; at += 65535) {
        const int64_t rows = std::min<int64_t>(batch - at, 65535);
        Args a{*q, *k, *v, log_decay, state, slots ? slots + at : nullptr, nullptr, pool, dk, dv, scale};
        a.q.data = static_cast<const char*>(q->data) + at * q->batch_stride * elem;
        a.k.data = static_cast<const char*>(k->data) + at * k->batch_stride * elem;
        a.v.data = static_cast<const char*>(v->data) + at * v->batch_stride * elem;
        a.o = static_cast<char*>(o) + at * q->heads * dv * elem;
        if (!slots) a.state = state + at * k->heads * int64_t(dk) * dv, a.pool = pool - at;
        if (dtype == FCQT_F32) launch<float>(a, rows, stream);
        else if (dtype == FCQT_BF16) launch<bf16>(a, rows, stream);
        else launch<f16>(a, rows, stream);
        if (int e = launched()) return e;
    }
    return FCQT_OK;
}
