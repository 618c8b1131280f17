// Linear attention with a decay for each head, over whole sequences, on matrix instructions.
//
//   S_t = e^g S_{t-1} + k_t v_t',   o_t = scale q_t S_t
//
// in chunks of C tokens, n of them valid. With X the state before a chunk and L = e^g,
//   o_i = L^(i+a) q_i X + sum over j <= i of L^(i-j) (q_i k_j) v_j
//   X  <- L^n X + sum over j of L^(n-a-j) k_j v_j'                        (a = 1)
// The gradients are the same operator with its operands exchanged:
//   dq = A(do, v, k) with S';  dv = A(k, q, do) and dk = A(v, do, q) back in time (a = 0), with S's gradient.
// The slope by g is the sum of (t - s) c(s, t) over pairs of tokens. With Z the state's gradient after a chunk, dq and dk
// without the products inside the chunk (those from X and from Z), a chunk gives
//   sum of (i+1) <q_i, dq_i> + sum of (n-1-j) <k_j, dk_j> + n L^n <X, Z>
//     + sum over j <= i of (i-j) L^(i-j) (do_i v_j) (q_i k_j)
// : pairs that end in it, begin in it, cross it and lie in it, no differences of large sums. (Without <X, Z> the flow
// of c past each chunk would follow from sums of <q, dq> - <k, dk>, which lose a factor of 10 and more for a head that
// remembers few tokens.) dk's kernel (kSlope 2) leaves its state at every chunk's end for dq's (kSlope 1), which needs
// both: an element is written and read once for each chunk of tokens, as many bytes as q, k, v and do hold.
//
// One workgroup walks a segment of one (row, key head) from its first to its last chunk with the state in registers:
// wave w owns 32 columns of it, all KD rows, as accumulators of v_mfma_f32_32x32x16_bf16. The layouts fit without any
// exchange between lanes: an accumulator tile's registers hold, in order, what the B operand (state) or A operand (P')
// of the next product wants once the products' inner index is taken in the order 0-3, 8-11 | 4-7, 12-15, which the
// tiles of q and k are stored in. Operands whose inner index is the token are read with the transposing LDS load.
//
// Precision: bf16 inputs are exact operands, fp16 ones two planes, and fp32 ones and what is computed (P, the state, the
// decayed v) three bf16 planes whose sum is the fp32 value: six bf16 products for one fp32 product take 192 cycles where
// v_mfma_f32_32x32x2_f32 takes 512. (Two planes for what 16-bit outputs are made of would leave 2^-17 of each operand, and
// o 1.3e-6 of its size away from its value before the rounding, where three leave 2e-7.)
//
// What bounds it: 1 x 65537 bf16 tokens of 16 heads, 128 wide, take 373 us in the main kernel (1.11 GB, 3.0 TB/s) after
// 128 us for the segments' own states (0.54 GB, 4.2 TB/s): about 1600 vector and 136 matrix instructions a wave and chunk,
// 169 and 117 us of the SIMDs' time; the rest is waiting for LDS, barriers and products that need each other, which two
// waves a SIMD (their registers are full of state) cover in part. Every wave computes all of P, whose rows its columns of v
// need. A pass of one segment would need no states first, but 16 workgroups leave 240 compute units idle. 8 x 512 fp32
// tokens of 8 heads of 64: 15 us, 12 for the states, 5 between them, each little more than its launch and one chunk after
// the other. dq's kernel with the slope's terms takes 198 us for 9 rows of 0 to 4097 tokens, 16 heads on 8 (dq alone 115, dk
// with its half of the terms 158): most of the difference is the states at the chunks' ends, 64 KB for 64 tokens of a head.
// fp16's two planes and 32-token chunks take 573 us where bf16 takes 373.
// Chunks of 64 tokens, or of 32 where planes take the LDS: at 32 tokens bf16 would read twice as many of those.
#pragma once

#include <type_traits>

#include "seq_common.hpp"

namespace fcqt_seq {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f32x2 = float __attribute__((ext_vector_type(2)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using i16x4 = short __attribute__((ext_vector_type(4)));

// a state tensor: element (row, col) of head h, batch row b, segment s
struct State {
    float* data;
    int64_t batch, head, segment;
    int32_t row, col;
    __device__ float* at(int64_t b, int h, int s) const { return data + b * batch + h * head + s * segment; }
};

struct Chunks {
    fcqt_heads q, k, v;
    const float* log_decay;
    const int32_t* lengths;        // or NULL: all tokens
    State first, last;             // states before each segment; states after (of segments, or of the whole)
    // the slope by g: what the output is multiplied with, the state's gradients at the chunks' ends (as the registers
    // hold them), sums [batch][heads (query heads: spread)][segments][waves]
    fcqt_heads w;
    float* flow;
    double* slopes;
    void* o;                       // [batch][tokens][output heads][vd]
    int64_t tokens;
    int32_t kd, vd, group;         // group: query heads of a key head
    int32_t segments, chunks;      // chunks of a segment
    int32_t back, reduce;          // back: from the last token to the first; reduce: the group is on k's and v's side
    int32_t spread;                // every query head has a workgroup of its own (not with reduce)
    float p_scale, u_scale, x_scale;   // of P, of what enters the state, of what comes from it
};

// Tokens of a chunk: 64, or 32 where the inputs' planes take the LDS.
constexpr int chunk_tokens(int planes) { return planes == 1 ? 64 : 32; }

// Sizes of one kernel. NI: planes of an input; C: tokens of a chunk.
// kRows: v's rows are operands too.
template <int NI, int KD, int NW, bool kRows = false>
struct Tile {
    static constexpr int C = chunk_tokens(NI);
    static constexpr int threads = 64 * NW;
    // Rows of q and k: 80 bytes of padding make both their reads fall on different banks (16 rows of 16 bytes; 4 rows
    // of 64 bytes in the transposing read, all but a few). Rows of v: 64 bytes for the latter alone.
    static constexpr int krow = KD + 40, vrow = 32 * NW + (kRows ? 40 : 32);
    static constexpr int kplane = C * krow, vplane = C * vrow;
    // groups of 8 elements of a tile, and how many of them a thread stages
    static constexpr int kgroups = C * KD / 8, vgroups = C * 4 * NW;
    static constexpr int nk = (kgroups + threads - 1) / threads, nv = vgroups / threads;
};

template <class T>
struct Planes;
template <>
struct Planes<bf16> { static constexpr int n = 1; };
template <>
struct Planes<f16> { static constexpr int n = 2; };
template <>
struct Planes<float> { static constexpr int n = 3; };

__device__ __forceinline__ bf16x2 pair(float a, float b) {
    return __builtin_convertvector(f32x2{a, b}, bf16x2);
}

// x as the sum of N planes, each the nearest bf16 of what the ones before leave
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&y)[N]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int p = 0; p < N; ++p) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const bf16x2 t = pair(r[e], r[e + 1]);
            y[p][e] = t[0];
            y[p][e + 1] = t[1];
            if (p + 1 < N) {
                r[e] -= float(t[0]);
                r[e + 1] -= float(t[1]);
            }
        }
    }
}

// acc += a b over the planes whose product counts (of order two and below: the others are under 2^-24), the small ones first
template <int NA, int NB>
__device__ __forceinline__ void multiply(f32x16& acc, const bf16x8 (&a)[NA], const bf16x8 (&b)[NB]) {
#pragma unroll
    for (int order = 2; order >= 0; --order)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (order - i >= 0 && order - i < NB) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[order - i], acc, 0, 0, 0);
}

constexpr int kPlanes = 3;          // of what is computed

// eight input elements as they lie in memory
template <class T>
struct alignas(16) Raw {
    T e[8];
};

// Four tokens of a column in each of two blocks: the transposing load of a 4 x 16 block, its rows `stride` elements
// apart; `p` is this lane's quarter row.
__device__ __forceinline__ bf16x8 transposed(const uint16_t* p, int second) {
    using as3 = __attribute__((address_space(3))) i16x4*;
    const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((as3)(p));
    const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((as3)(p + second));
    using i16x8 = short __attribute__((ext_vector_type(8)));
    const i16x8 c = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, c);
}

// keeps the compiler from moving loads (whose registers are the state's) and products over this place
__device__ __forceinline__ void fence() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// a value that all lanes hold, in a scalar register
__device__ __forceinline__ float uniform(float x) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// L^n. The exponent's rounding, which would put the same error on all of a distance's terms, is made good: expf(x + e).
__device__ __forceinline__ float power(float g, int n) {
    if (n == 0) return 1.0f;
    const float x = g * float(n), y = expf(x);
    return fabsf(x) < 100.0f ? fmaf(y, fmaf(g, float(n), -x), y) : y;
}

// What n tokens make of a state that goes on: near one L^n itself, rounded, would be off by the same amount at every chunk,
// segment or call of as many tokens, which adds up over a head's horizon (6000 calls of one token, g = -1e-4: 6e-5 of the
// state), so L^n x is x + expm1(g n) x in one rounding there.
struct Decay {
    bool slow;
    float by;                       // expm1(g n) or, for large n, L^n
    __device__ __forceinline__ Decay(float g, int n) : slow(g * float(n) > -0.5f), by(slow ? expm1f(g * float(n)) : power(g, n)) {}
};

// kStates: states alone, no output. kSlope: with the slope's terms (1 of dq, 2 of dk). Its registers are shared among two
// waves of a SIMD.
template <class T, int KD, int NW, bool kStates, int kSlope>
__global__ __launch_bounds__(64 * NW, 2) void k_chunks(Chunks a) {
    constexpr int NI = Planes<T>::n;
    using Z = Tile<NI, KD, NW, kSlope == 1>;
    constexpr int C = Z::C, NT = Z::threads, IT = C / 32, MT = KD / 32, TILES = IT * (IT + 1) / 2;
    constexpr int E = 16 / sizeof(T);                                // elements of 16 bytes
    // the compiler is kept from hoisting the loads of many steps: their registers are the state's
    constexpr int kFence = NI == 1 ? 2 : 1;
    // one object: the places in it differ by constants, and a lane's offset serves them all
    __shared__ struct __attribute__((aligned(16))) {
        uint16_t q[kStates ? 8 : NI * Z::kplane], k[NI * Z::kplane], v[NI * Z::vplane];
        // powers of the decay: of i - j at C - 1 - i + j (zero where j > i), of a query's, of a token's in the state
        float near[2 * C], ahead[C], left[C];
        T o[kStates ? 1 : NW][kStates ? 16 : 32][32 + E];                // a wave's outputs on their way
    } lds;
    uint16_t *const qs = lds.q, *const ks = lds.k, *const vs = lds.v;
    float *const near = lds.near, *const ahead = lds.ahead, *const left = lds.left;

    // dq's kernel and dk's run one way each; the others both
    const bool back = kSlope ? kSlope == 2 : a.back != 0, reduce = kSlope == 2 || a.reduce != 0;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 32, half = lane / 32;
    const int seg = blockIdx.x;
    const int spread = kStates || reduce ? 0 : a.spread, head = __builtin_amdgcn_readfirstlane(spread ? blockIdx.y / a.group : blockIdx.y);
    const int own = spread ? blockIdx.y - head * a.group : 0, keys = reduce ? a.q.heads : a.k.heads;
    const int64_t row = blockIdx.z;
    const int vcol = wave * 32 + col;              // this lane's column of the state
    const bool vin = vcol < a.vd;
    const float g = a.log_decay[head];
    const int shift = back ? 0 : 1;                                // the a of the formulas
    const int64_t length = a.lengths ? min(max(int64_t(a.lengths[row]), int64_t(0)), a.tokens) : a.tokens;
    const int64_t begin = int64_t(seg) * a.chunks * C;
    const int64_t end = min(begin + int64_t(a.chunks) * C, a.tokens);

    for (int x = threadIdx.x; x < 2 * C; x += NT) {
        const int n = C - 1 - x;
        near[x] = n < 0 ? 0.0f : a.p_scale * power(g, n);
        if (x < C) ahead[x] = a.x_scale * power(g, x + shift);
    }

    f32x16 S[MT];
    // Addresses are a uniform base and a 32-bit offset of the lane's (the host checks that a chunk's rows and a state
    // lie within 2^31 bytes): 64-bit ones of every access would take the registers that the state is kept in.
    // `hidden` keeps the compiler from carrying one use's offsets over the whole loop to the next.
    auto hidden = [](int x) {
        asm volatile("" : "+v"(x));
        return x;
    };
    auto offset = [&](const State& s, int h, int c, int m, int r) {
        const int k = m * 32 + 8 * (r / 4) + 4 * h + r % 4;
        return k < a.kd && c < a.vd ? k * s.row + c * s.col : -1;
    };
    auto read_state = [&](const State& s, f32x16* X) {
        if (!s.data) {
#pragma unroll
            for (int m = 0; m < MT; ++m) X[m] = f32x16{};
            return;
        }
        const float* base = s.at(row, head, seg);
        const int h = hidden(half), c = hidden(vcol);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int at = offset(s, h, c, m, r);
                const float x = base[uint32_t(max(at, 0))];
                X[m][r] = at < 0 ? 0.0f : x;
            }
    };
    auto write_state = [&](const State& s, const f32x16* X) {
        float* base = s.at(row, head, seg);
        const int tid = hidden(threadIdx.x), h = tid / 32 % 2, c = tid / 64 * 32 + tid % 32;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int at = offset(s, h, c, m, r);
                if (at >= 0) base[uint32_t(at)] = X[m][r];
            }
    };
    read_state(a.first, S);

    // What is staged: groups of eight elements in registers while the chunk before is computed. Groups that are not
    // there (rows past n, columns past dim) are loaded from the first row's first group and staged as zeros.
    Raw<T> rq[kStates ? 1 : Z::nk], rk[Z::nk], rv[Z::nv];
    auto fetch = [&]<int count, int width>(Raw<T> (&to)[count], std::integral_constant<int, width>, const fcqt_heads& s, int h,
                                           int64_t c0, int n, int dim) {
        const char* p = reinterpret_cast<const char*>(static_cast<const T*>(s.data) + row * s.batch_stride + h * s.head_stride + c0 * s.token_stride);
        const uint32_t stride = uint32_t(s.token_stride) * sizeof(T);
        constexpr int across = width / 8, down = NT / across;
        static_assert(NT % across == 0);
        const int tid = hidden(threadIdx.x), r0 = tid / across, c = tid % across * 8;
#pragma unroll
        for (int i = 0; i < count; ++i) {
            const int r = r0 + i * down;
            const uint32_t t = back ? n - 1 - r : r;
            const uint32_t at = r < n && c < dim ? t * stride + uint32_t(c) * sizeof(T) : 0u;
            to[i] = *reinterpret_cast<const Raw<T>*>(p + at);
        }
    };
    auto planes_of = [&](const Raw<T>& x, bool in, bf16x8 (&y)[NI]) {
        if constexpr (NI == 1) {
            y[0] = __builtin_bit_cast(bf16x8, x);
            if (!in) y[0] = bf16x8{};
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = in ? widen<T>(x.e[e]) : 0.0f;
            split<NI>(f, y);
        }
    };
    auto stage_k = [&](const Raw<T>* from, uint16_t* to, int n, auto whole) {
        const int tid = hidden(threadIdx.x), r0 = tid / (KD / 8), c = tid % (KD / 8);
#pragma unroll
        for (int i = 0; i < Z::nk; ++i) {
            const int r = r0 + i * (NT / (KD / 8));
            if (Z::kgroups % NT && r >= C) continue;
            bf16x8 y[NI];
            planes_of(from[i], whole || (r < n && c * 8 < a.kd), y);
#pragma unroll
            for (int p = 0; p < NI; ++p) {
                uint16_t* at = to + p * Z::kplane + r * Z::krow + c / 2 * 16 + c % 2 * 4;
                const uint4 u = __builtin_bit_cast(uint4, y[p]);
                *reinterpret_cast<uint2*>(at) = make_uint2(u.x, u.y);
                *reinterpret_cast<uint2*>(at + 8) = make_uint2(u.z, u.w);
            }
        }
    };
    auto stage_v = [&](const Raw<T>* from, uint16_t* to, int n, auto whole) {
        const int tid = hidden(threadIdx.x), r0 = tid / (4 * NW), c = tid % (4 * NW);
#pragma unroll
        for (int i = 0; i < Z::nv; ++i) {
            const int r = r0 + i * (NT / (4 * NW));
            bf16x8 y[NI];
            planes_of(from[i], whole || (r < n && c * 8 < a.vd), y);
#pragma unroll
            for (int p = 0; p < NI; ++p) {
                if constexpr (kSlope == 1) {
                    uint16_t* at = to + p * Z::vplane + r * Z::vrow + c / 2 * 16 + c % 2 * 4;
                    const uint4 u = __builtin_bit_cast(uint4, y[p]);
                    *reinterpret_cast<uint2*>(at) = make_uint2(u.x, u.y);
                    *reinterpret_cast<uint2*>(at + 8) = make_uint2(u.z, u.w);
                } else {
                    *reinterpret_cast<bf16x8*>(to + p * Z::vplane + r * Z::vrow + c * 8) = y[p];
                }
            }
        }
    };

    // the segment's chunks that hold a valid token come first; a step is one of them with one head of the group
    const int live = int(max((min(length, end) - begin + C - 1) / C, int64_t(0)));
    const int per = spread || (kStates && !reduce) ? 1 : a.group, steps = live * per;
    auto chunk_at = [&](int i) { return begin + int64_t(back ? live - 1 - i : i) * C; };
    auto valid_of = [&](int64_t c0) { return int(min(min(length, end) - c0, int64_t(C))); };
    auto load = [&](int i, int gi) {
        const int64_t c0 = chunk_at(i);
        const int n = valid_of(c0), one = head * a.group + own + gi, h = reduce ? one : head;
        if constexpr (!kStates) fetch(rq, std::integral_constant<int, KD>{}, a.q, reduce ? head : one, c0, n, a.kd);
        fetch(rk, std::integral_constant<int, KD>{}, a.k, h, c0, n, a.kd);
        fetch(rv, std::integral_constant<int, 32 * NW>{}, a.v, h, c0, n, a.vd);
    };

    // places of this lane in the tiles
    const uint16_t* qat = qs + col * Z::krow + half * 8;
    const uint16_t* kat = ks + col * Z::krow + half * 8;
    const int tr = lane % 16 / 4, tc = lane % 4, tb = lane / 16 % 2;
    const uint16_t* ktr = ks + (4 * half + tr) * Z::krow + tb * 16 + (tc % 2 * 8 + tc / 2 * 4);
    const uint16_t* vtr = vs + (4 * half + tr) * Z::vrow + wave * 32 + tb * 16 + (kSlope == 1 ? tc % 2 * 8 + tc / 2 * 4 : tc * 4);

    const bool fits = a.kd == KD && a.vd == 32 * NW;  // no columns that are not there
    f32x16 O[kStates ? 1 : IT];                                      // transposed: rows the columns of v, columns the queries
    double slopes = 0;                                               // (terms of both signs, far larger than their sum)
    int before = -1;                                                 // the n that `left` and the next two were made for
    float by = 0, same = 0;                                          // Decay: what the state gets and keeps of itself
    const int chunks = int((a.tokens + C - 1) / C);
    auto flow_at = [&](int64_t c0) {                                 // this wave's part of a chunk's state
        // (a count of pieces of 8 KB and more)
        const uint32_t at = ((uint32_t(row) * keys + head) * chunks + uint32_t(c0 / C));
        return reinterpret_cast<f32x4*>(a.flow) + int64_t(at) * (NW * MT * 256);
    };
    if (steps) load(0, 0);
    for (int step = 0, ci = 0, gi = 0; step < steps; ++step) {
        const int64_t c0 = chunk_at(ci);
        const int n = valid_of(c0);
        float slope = 0;
        const bool first = gi == 0, final = gi == per - 1, more = step + 1 < steps;
        const int ci1 = more && final ? ci + 1 : ci, gi1 = more ? (final ? 0 : gi + 1) : gi;
        const int oh = reduce ? head : head * a.group + own + gi, heads = a.q.heads;
        __syncthreads();
        auto stage = [&](auto whole) {
            if constexpr (!kStates) stage_k(rq, qs, n, whole);
            stage_k(rk, ks, n, whole);
            stage_v(rv, vs, n, whole);
        };
        if (n == C && fits) stage(std::true_type{});
        else stage(std::false_type{});
        if constexpr (kStates) {
            // what is left of the segment after a token: the state needs no decay on the way
            const int rest = int(back ? c0 - begin : min(length, end) - c0 - n);
            if (first) {
                for (int x = threadIdx.x; x < C; x += NT) left[x] = x < n ? a.u_scale * power(g, rest + n - shift - x) : 0.0f;
            }
        } else if (n != before) {
            for (int x = threadIdx.x; x < C; x += NT) {
                const int m = n - shift - x;
                left[x] = m < 0 ? 0.0f : a.u_scale * power(g, m);
            }
            const Decay f(g, n);
            by = uniform(f.by), same = uniform(f.slow ? 1.0f : 0.0f);
            before = n;
        }
        __syncthreads();
        // the next chunk's loads; where the slope's terms want their registers, later. Three planes' LDS leaves one wave a
        // SIMD, with registers for all of it.
        constexpr bool kEarly = kSlope == 0 || NI == 3;
        if (kEarly) load(ci1, gi1);
        if constexpr (kSlope == 2) {
            if (first) {
                f32x4* at = flow_at(c0);
                const uint32_t here = hidden(wave * MT * 256 + lane);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < 4; ++r) at[here + uint32_t((m * 4 + r) * 64)] = f32x4{S[m][4 * r], S[m][4 * r + 1], S[m][4 * r + 2], S[m][4 * r + 3]};
            }
        }
        // a tile's rows of w as the output's registers lie, zeros past n
        using Four = uint32_t __attribute__((ext_vector_type(sizeof(T))));     // four elements
        Four w[kSlope == 1 ? IT : 1][4];
        auto load_w = [&](int i, Four (&to)[4]) {
            const int columns = min(a.vd - wave * 32, 32);
            const char* p = reinterpret_cast<const char*>(static_cast<const T*>(a.w.data) + row * a.w.batch_stride + oh * a.w.head_stride + c0 * a.w.token_stride + (columns > 0 ? wave * 32 : 0));
            const int h = hidden(half), r = i * 32 + hidden(col);
            const uint32_t t = back ? n - 1 - r : r;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int c = 8 * x + 4 * h;
                const bool in = r < n && c < columns;
                const Four y = *reinterpret_cast<const Four*>(p + (in ? t * uint32_t(a.w.token_stride) + uint32_t(c) : 0u) * sizeof(T));
                to[x] = in ? y : Four(0u);
            }
        };
        // columns 16 s to 16 s + 15 of it as an operand
        auto rows_of = [&](const Four (&w)[4], int s, bf16x8 (&y)[NI]) {
            if constexpr (NI == 1) {
                y[0] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(w[2 * s], w[2 * s + 1], 0, 1, 2, 3));
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const Four u = w[2 * s + e / 4];
                    if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(u[e % 4]);
                    else x[e] = widen<T>(T{uint16_t(u[e % 4 / 2] >> (e % 2 * 16))});
                }
                split<NI>(x, y);
            }
        };
        auto dot = [&](const Four (&w)[4], const f32x16& x) {
            float sum = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const Four y = w[r / 4];
                if constexpr (sizeof(T) == 4) sum += x[r] * __uint_as_float(y[r % 4]);
                else sum += x[r] * widen<T>(T{uint16_t(y[r % 4 / 2] >> (r % 2 * 16))});
            }
            return sum;
        };
        if constexpr (kSlope == 1) {
#pragma unroll
            for (int i = 0; i < IT; ++i) load_w(i, w[i]);
        }
        float crossing = 0;
        f32x16 A[kStates ? 1 : TILES];
        // the last tile's products when they are wanted: their registers hold w's rows until then
        constexpr bool kLater = kSlope == 1 && IT > 1;
        if constexpr (!kStates) {
            // O' = X' q' and P' = k q' of all tiles with j <= i (kLater: of j = 0), from one read of q and k
            // Between them, n L^n <X, Z> (kSlope 1, with a group's last head): 16 rows of Z are on their way while X's are
            // multiplied.
            const bool crosses = kSlope == 1 && final && own == 0;
            constexpr int kAhead = NI == 3 ? KD / 16 : 1;                  // one wave a SIMD has registers for all of it
            f32x4 z[kAhead][2];
            auto load_z = [&](int s) {
                const f32x4* at = flow_at(c0);
                const uint32_t here = hidden(wave * MT * 256 + lane);
#pragma unroll
                for (int r = 0; r < 2; ++r) z[s % kAhead][r] = at[here + uint32_t((s * 2 + r) * 64)];
            };
            if constexpr (kSlope == 1 && kAhead > 1) {
                if (crosses) {
#pragma unroll
                    for (int s = 0; s < kAhead; ++s) load_z(s);
                }
            }
            auto inner = [&](auto inter) {
#pragma unroll
                for (int s = 0; s < KD / 16; ++s) {
                    if constexpr (kSlope == 1 && inter) {
                        if (crosses && kAhead == 1) load_z(s);
                    }
                    bf16x8 Q[IT][NI], K[NI], X[kPlanes];
#pragma unroll
                    for (int i = 0; i < IT; ++i)
#pragma unroll
                        for (int p = 0; p < NI; ++p) Q[i][p] = *reinterpret_cast<const bf16x8*>(qat + p * Z::kplane + i * 32 * Z::krow + s * 16);
                    if constexpr (inter) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = S[s / 2][8 * (s % 2) + e];
                        split<kPlanes>(x, X);
#pragma unroll
                        for (int i = 0; i < IT; ++i) multiply(O[i], X, Q[i]);
                    }
#pragma unroll
                    for (int j = 0; j < (kLater ? 1 : IT); ++j) {
#pragma unroll
                        for (int p = 0; p < NI; ++p) K[p] = *reinterpret_cast<const bf16x8*>(kat + p * Z::kplane + j * 32 * Z::krow + s * 16);
#pragma unroll
                        for (int i = j; i < IT; ++i) multiply(A[i * (i + 1) / 2 + j], K, Q[i]);
                    }
                    if constexpr (kSlope == 1 && inter) {
                        if (crosses) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) crossing += z[s % kAhead][e / 4][e % 4] * S[s / 2][8 * (s % 2) + e];
                        }
                    }
                    if (s % kFence == kFence - 1) fence();
                }
            };
#pragma unroll
            for (int t = 0; t < TILES; ++t) A[t] = f32x16{};
            if (!reduce || first) {
#pragma unroll
                for (int i = 0; i < IT; ++i) O[i] = f32x16{};
                inner(std::true_type{});
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const float f = ahead[i * 32 + hidden(col)];
#pragma unroll
                    for (int r = 0; r < 16; ++r) O[i][r] *= f;
                }
            } else {
                inner(std::false_type{});
            }
        }
        if (!kEarly && kSlope == 2) load(ci1, gi1);
        const bool decays = !kStates && (reduce ? first : final), updates = (reduce || kStates || final) && (kStates || a.last.data || step + per < steps);
        if (decays) {
            if constexpr (kSlope == 1) slope += (by + same) * float(n) * crossing;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[m][r] = fmaf(by, S[m][r], same * S[m][r]);
        }
        fence();
#pragma unroll
        for (int j = 0; j < IT; ++j) {
            bf16x8 V[2][NI];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int p = 0; p < NI; ++p)
                    V[s][p] = transposed(vtr + p * Z::vplane + (j * 32 + s * 16) * Z::vrow, 8 * Z::vrow);
            if constexpr (kLater) {
                if (j) {
                    static_assert(IT <= 2);
#pragma unroll
                    for (int s = 0; s < KD / 16; ++s) {
                        bf16x8 Q[NI], K[NI];
#pragma unroll
                        for (int p = 0; p < NI; ++p) {
                            Q[p] = *reinterpret_cast<const bf16x8*>(qat + p * Z::kplane + j * 32 * Z::krow + s * 16);
                            K[p] = *reinterpret_cast<const bf16x8*>(kat + p * Z::kplane + j * 32 * Z::krow + s * 16);
                        }
                        multiply(A[TILES - 1], K, Q);
                        if (s % kFence == kFence - 1) fence();
                    }
                }
            }
            if constexpr (!kStates) {
#pragma unroll
                for (int i = j; i < IT; ++i) {
                    constexpr int kw = kSlope == 1 ? 1 : 0;
                    if (kSlope == 2 && j == 0 && first) load_w(i, w[0]);
                    if (kSlope && j == 0 && (!reduce || first)) {
                        slope += dot(w[i * kw], O[i]) * float(i * 32 + hidden(col) + shift);
                    }
                    // of the rows of w and v in this wave's columns: the products of queries and keys that the slope wants
                    f32x16 B{};
                    if constexpr (kSlope == 1) {
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            bf16x8 W[NI], R[NI];
                            rows_of(w[i * kw], s, W);
#pragma unroll
                            for (int p = 0; p < NI; ++p) R[p] = *reinterpret_cast<const bf16x8*>(vs + hidden(col) * Z::vrow + wave * 32 + hidden(half) * 8 + p * Z::vplane + j * 32 * Z::vrow + s * 16);
                            multiply(B, R, W);
                        }
                        fence();
                    }
                    const int x0 = C - 1 - i * 32 - hidden(col) + j * 32 + 4 * hidden(half);
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        float x[8];
                        bf16x8 P[kPlanes];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = A[i * (i + 1) / 2 + j][8 * s + e] * near[x0 + 8 * (2 * s + e / 4) + e % 4];
                        split<kPlanes>(x, P);
                        multiply(O[i], V[s], P);
                        if constexpr (kSlope == 1) {
                            const float d = float(hidden(i * 32 + col - j * 32 - 4 * half));
#pragma unroll
                            for (int e = 0; e < 8; ++e) slope += (d - float(8 * (2 * s + e / 4) + e % 4)) * x[e] * B[8 * s + e];
                        }
                    }
                    fence();
                }
            }
            if (!updates) continue;
            // X += k' (L^(n-a-j) v)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float x[8];
                bf16x8 W[kPlanes];
                const f32x4 f0 = *reinterpret_cast<const f32x4*>(&left[j * 32 + s * 16 + 4 * half]);
                const f32x4 f1 = *reinterpret_cast<const f32x4*>(&left[j * 32 + s * 16 + 8 + 4 * half]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float v = float(V[s][NI - 1][e]);
#pragma unroll
                    for (int p = NI - 2; p >= 0; --p) v += float(V[s][p][e]);
                    x[e] = v * (e < 4 ? f0[e % 4] : f1[e % 4]);
                }
                split<kPlanes>(x, W);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    bf16x8 K[NI];
#pragma unroll
                    for (int p = 0; p < NI; ++p)
                        K[p] = transposed(ktr + p * Z::kplane + (j * 32 + s * 16) * Z::krow + m * 32, 8 * Z::krow);
                    multiply(S[m], K, W);
                    if (m % 2) fence();
                }
                fence();
            }
        }
        if (!kEarly && kSlope == 1) load(ci1, gi1);
        if constexpr (!kStates) {
            if (!reduce || final) {
                const int rows = int(min(int64_t(C), end - c0));
                char* out = reinterpret_cast<char*>(static_cast<T*>(a.o) + ((row * a.tokens + c0) * heads + oh) * a.vd + hidden(threadIdx.x) / 64 * 32);
                const uint32_t ostride = uint32_t(heads * a.vd) * sizeof(T);
                const int columns = min(a.vd - wave * 32, 32);     // of this wave's
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    // through LDS, in which a token's 32 values come together
                    T* mine = &lds.o[wave][hidden(col)][4 * hidden(half)];
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const float y[4] = {O[i][r], O[i][r + 1], O[i][r + 2], O[i][r + 3]};
                        store<T, 4>(mine + 2 * r, y);
                    }
                    __builtin_amdgcn_wave_barrier();
                    constexpr int across = 32 / E, down = 64 / across;
                    const int l = hidden(lane), c = l % across * E;
#pragma unroll
                    for (int x = 0; x < 32; x += down) {
                        const int at = x + l / across, r = i * 32 + at;
                        uint4 y = *reinterpret_cast<const uint4*>(&lds.o[wave][at][c]);
                        if (r >= n) y = uint4{};
                        const uint32_t t = back && r < n ? n - 1 - r : r;
                        if (r < rows && c < columns) *reinterpret_cast<uint4*>(out + (t * ostride + uint32_t(c) * sizeof(T))) = y;
                    }
                    __builtin_amdgcn_wave_barrier();
                }
            }
        }
        if constexpr (kSlope != 0) slopes += slope;
        ci = ci1, gi = gi1;
    }
    if constexpr (!kStates) {                                        // past the row's end
        const int group = reduce || spread ? 1 : a.group, across = a.vd / E;
        const int64_t t0 = begin + int64_t(live) * C;
        T* out = static_cast<T*>(a.o) + (row * a.tokens * a.q.heads + (reduce ? head : head * a.group + own)) * a.vd;
        for (int64_t x = threadIdx.x; x < (end - t0) * group * across; x += NT) {
            const int64_t y = x / across, t = t0 + y / group;
            *reinterpret_cast<uint4*>(out + (t * a.q.heads + y % group) * a.vd + x % across * E) = uint4{};
        }
    }
    if (kStates || (a.last.data && own == 0 && seg == (back ? 0 : a.segments - 1))) write_state(a.last, S);
    if constexpr (kSlope != 0) {
#pragma unroll
        for (int d = 32; d; d /= 2) slopes += __shfl_xor(slopes, d);
        if (lane == 0) {
            a.slopes[((row * gridDim.y + blockIdx.y) * a.segments + seg) * NW + hidden(threadIdx.x) / 64] = slopes;
        }
    }
}

// Which kernel, and over what. grid: segments, key heads (or query heads), rows.
struct Launch {
    int kd, waves;                  // the kernel's sizes: 32, 64 or 128, 2 or 4
    bool states;                    // states alone
    int slope;                      // kSlope
    dim3 grid;
    hipStream_t stream;
};

template <class T, int KD, int NW>
void launch_sized(const Chunks& a, const Launch& l) {
    if (l.states) k_chunks<T, KD, NW, true, 0><<<l.grid, 64 * NW, 0, l.stream>>>(a);
    else if (l.slope == 1) k_chunks<T, KD, NW, false, 1><<<l.grid, 64 * NW, 0, l.stream>>>(a);
    else if (l.slope == 2) k_chunks<T, KD, NW, false, 2><<<l.grid, 64 * NW, 0, l.stream>>>(a);
    else k_chunks<T, KD, NW, false, 0><<<l.grid, 64 * NW, 0, l.stream>>>(a);
}

template <class T>
void launch_kind(const Chunks& a, const Launch& l) {
    switch (l.kd * 8 + l.waves) {
        case 32 * 8 + 2: return launch_sized<T, 32, 2>(a, l);
        case 32 * 8 + 4: return launch_sized<T, 32, 4>(a, l);
        case 64 * 8 + 2: return launch_sized<T, 64, 2>(a, l);
        case 64 * 8 + 4: return launch_sized<T, 64, 4>(a, l);
        case 128 * 8 + 2: return launch_sized<T, 128, 2>(a, l);
        default: return launch_sized<T, 128, 4>(a, l);
    }
}

// one source file for each type
void launch_f32(const Chunks& a, const Launch& l);
void launch_bf16(const Chunks& a, const Launch& l);
void launch_f16(const Chunks& a, const Launch& l);

}  // namespace fcqt_seq
