// One AdamW step over many tensors, and reading 8-bit moments back.
//
//   m = b1 m + c1 g,  v = b2 v + c2 g g,  p = keep p - rate m / (root sqrt(v) + eps)
//
// Every product and sum is rounded on its own (no fused multiply-add), so the step gives the bits that a chain of
// elementwise fp32 operations gives, and 8-bit codes do not depend on how a compiler pairs operations.
//
// 8-bit moments: FCQT_ADAMW_BLOCK elements share one fp32 scale, their largest magnitude over 1.9375. A code is a
// small float of four mantissa bits: m has a sign bit and three exponent bits, sqrt(v) (which is held instead of v:
// half the range in exponents) four exponent bits. A code's value comes out of shifts alone, no table. sqrt(v) > 0
// never becomes code 0: a vanished spread would leave m / eps.
//
// A code is the nearest one, or (fcqt_adamw_drawn) one of the two neighbours, drawn so that m and v are kept on average.
// The nearest serves a single step; over many it is wrong: a step with b2 = 0.999 takes at most 0.05% off sqrt(v), far from
// half a code's step of 1.6 to 3.1%, so codes stay where they are. (1000 steps of unit noise leave v 1.3 of its value, drawn
// codes 1.00; 6000 steps after gradients fell to a tenth sqrt(v) is 9 times too large, drawn 0.99, 11 to 13% off (rms).)
// The draw is a hash of seed, step, tensor and element: the same call gives the same codes. v's chance is that of w w, not
// of w = sqrt(v), whose square would grow by the codes' variance (2% in all). Under m's smallest code the draw takes place
// where that code is a step of at most four learning rates (a gradient's own is up to (1 - b1) / sqrt(1 - b2), 3.2);
// beyond, m becomes zero: an element under 2^-13 of its block's moves by its gradients alone, where the draw would be rare
// steps of thousands of learning rates.
//
// Bound by memory with fp32 moments: 28 bytes an element with fp32 weights, 100 million in 512 us (5.5 TB/s; a copy 4.8).
// With 8-bit moments and bf16 weights 10 bytes an element; 100 million take 237 us (4.2 TB/s), about 100 instructions an element
// (exact quotients and roots) beside them, drawn codes 297 (the hash: three products an element at a quarter of the rate), and
// reading them back 150 (5.4 TB/s).
#include <algorithm>
#include <type_traits>

#include "seq_common.hpp"

using namespace fcqt_seq;

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = FCQT_ADAMW_BLOCK;
// tensors of one launch: their descriptors travel in the kernel's arguments (4 KB at most), so a step copies no
// table to the GPU and can be captured
constexpr int kMost = 56;

struct Tensors {
    fcqt_adamw_tensor t[kMost];
    uint32_t first[kMost];     // first workgroup of each tensor
    int count;
};

// what the draws of each tensor start from
template <bool kDraw>
struct Keys {
    uint64_t of[kDraw ? kMost : 1];
};
static_assert(sizeof(Tensors) + sizeof(fcqt_adamw_factors) + sizeof(Keys<true>) + 32 <= 4096, "kernel arguments");

// A bijection of 64 bits whose every output bit depends on all input bits: products with odd numbers (of the golden ratio's
// and the root of three's digits) carry upwards, shifts downwards.
uint64_t mixed(uint64_t x) {
    x ^= x >> 32;
    x *= 0x9E3779B97F4A7C15ull;
    x ^= x >> 29;
    x *= 0xBB67AE8584CAA73Bull;
    return x ^ x >> 32;
}

// Two numbers in [0, 1) for element i of a tensor, by the same means in 32 bits.
__device__ __forceinline__ void drawn(uint64_t key, int64_t i, float& a, float& b) {
    uint32_t x = uint32_t(i) ^ uint32_t(key) ^ uint32_t(i >> 32) * 0x85D4A0ADu;
    x ^= x >> 16;
    x *= 0x9E3779B1u;
    x ^= uint32_t(key >> 32);
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    x ^= x >> 16;
    b = float(x >> 8) * 0x1p-24f;
    a = float(x * 0x9E3779B1u >> 8) * 0x1p-24f;
}

// the tensor that a workgroup works on
__device__ __forceinline__ int owner(const Tensors& a, uint32_t block) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float updated(float p, float g, float& m, float& v, float& w, const fcqt_adamw_factors& f) {
#pragma clang fp contract(off)
    const float m1 = m * f.b1, m2 = g * f.c1;
    m = m1 + m2;
    const float v1 = v * f.b2, v2 = g * f.c2;
    const float v3 = v2 * g;
    v = v1 + v3;
    w = sqrtf(v);
    const float root = w * f.root;
    const float step = m / (root + f.eps) * f.rate;
    return p * f.keep - step;
}

// ---------------------------------------------------------------- 8-bit codes

template <bool kUnsigned>
struct Code {
    static constexpr int low = kUnsigned ? 14 : 6;      // smallest normal magnitude 2^-low
    static constexpr int bias = kUnsigned ? 112 : 120;  // fp32's exponent bias less the code's

    // Read as the top of an fp32 number's fields, a code is its value times 2^-bias, below the normal range too (fp32's own
    // subnormal numbers): two exact products and one rounding, by the scale.
    static __device__ __forceinline__ float value(uint32_t c, float scale) {
#pragma clang fp contract(off)
        const uint32_t bits = kUnsigned ? c << 19 : (c & 127) << 19 | (c & 128) << 24;
        return __uint_as_float(bits) * __uint_as_float(uint32_t(127 + bias) << 23) * scale;
    }

    // inverse: 1 / scale. kNear: with a scale from 2^-70 to 2^100, where the quotient's remainder is an fp32 number (or the
    // code 0): a neighbour of the quotient, made good by its remainder times the rounded inverse, is the rounded quotient
    // (Markstein's theorem), in five instructions instead of eleven. kDraw: the code below or the one above, by the number r
    // in [0, 1); least: whether a first moment may become the smallest code.
    template <bool kNear, bool kDraw>
    static __device__ __forceinline__ uint32_t code(float x, float scale, float inverse, float r, bool least) {
#pragma clang fp contract(off)
        const float a = fabsf(x);
        float y;
        if constexpr (kNear) {
            float q = a * inverse;                                  // to two units in the last place
            q = fmaf(fmaf(-q, scale, a), inverse, q);               // to one
            y = fmaf(fmaf(-q, scale, a), inverse, q);
        } else {
            y = scale > 0 ? a / scale : 0.0f;
        }
        const uint32_t bits = __float_as_uint(y);
        const bool small = y < 1.0f / float(1 << low);
        const float units = y * float(1 << (low + 4));              // in the smallest codes' steps
        uint32_t c;
        if constexpr (kDraw) {
            const float whole = floorf(units);
            c = small ? uint32_t(int(whole)) : (bits >> 19) - (bias << 4);
            const float f = small ? units - whole : float(bits & 0x7FFFF) * 0x1p-19f;       // of the way to the next code
            if constexpr (kUnsigned) {
                // l and l + 1 (codes in steps of their binade): (l + f)^2 lies f (2 l + f) / (2 l + 1) of the way between squares
                const float twice = float(2 * (small ? c : 16 + (c & 15)));
                c += r * (twice + 1) < f * (twice + f);
            } else {
                c += r < f && (c || least);
            }
        } else {
            c = small ? uint32_t(int(rintf(units))) : ((bits + 0x3FFFF + ((bits >> 19) & 1)) >> 19) - (bias << 4);
        }
        if (kUnsigned) return a > 0 ? min(max(c, 1u), 255u) : 0u;
        return min(c, 127u) | (x < 0 ? 128u : 0u);
    }
};

// ---------------------------------------------------------------- kernels

template <class T>
__global__ __launch_bounds__(kThreads) void k_adamw(Tensors a, fcqt_adamw_factors f, const float* grad_scale) {
    constexpr int V = 4, kShare = kThreads * V;
    const int i = owner(a, blockIdx.x);
    const fcqt_adamw_tensor& t = a.t[i];
    const int64_t at = int64_t(blockIdx.x - a.first[i]) * kShare + threadIdx.x * V;
    const int64_t left = t.n - at;
    if (left <= 0) return;
    const float gs = grad_scale ? *grad_scale : 1.0f;
    T* p = static_cast<T*>(t.p) + at;
    const T* g = static_cast<const T*>(t.g) + at;
    float *m = static_cast<float*>(t.m) + at, *v = static_cast<float*>(t.v) + at;
    const uintptr_t places = (reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) * (16 / (sizeof(T) * V)) |
                             reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
    if (left >= V && (places & 15) == 0) {
        float pp[V], gg[V], mm[V], vv[V], w;
        load<T, V>(p, pp);
        load<T, V>(g, gg);
        load<float, V>(m, mm);
        load<float, V>(v, vv);
#pragma unroll
        for (int e = 0; e < V; ++e) pp[e] = updated(pp[e], grad_scale ? gg[e] * gs : gg[e], mm[e], vv[e], w, f);
        store<T, V>(p, pp);
        store<float, V>(m, mm);
        store<float, V>(v, vv);
        return;
    }
    for (int e = 0; e < min(int64_t(V), left); ++e) {
        float mm = m[e], vv = v[e], w;
        const float gg = widen<T>(g[e]);
        p[e] = narrow<T>(updated(widen<T>(p[e]), grad_scale ? gg * gs : gg, mm, vv, w, f));
        m[e] = mm;
        v[e] = vv;
    }
}

// A lane holds eight elements, half a wave one block's scale.
template <class T, bool kDraw>
__global__ __launch_bounds__(kThreads) void k_adamw8(Tensors a, fcqt_adamw_factors f, const float* grad_scale, Keys<kDraw> keys) {
#pragma clang fp contract(off)
    constexpr int V = 8, kShare = kThreads * V;
    const int i = owner(a, blockIdx.x);
    const fcqt_adamw_tensor& t = a.t[i];
    const int64_t at = int64_t(blockIdx.x - a.first[i]) * kShare + threadIdx.x * V;
    const int64_t left = t.n - at;
    const float gs = grad_scale ? *grad_scale : 1.0f;
    T* p = static_cast<T*>(t.p) + at;
    const T* g = static_cast<const T*>(t.g) + at;
    uint8_t *m = static_cast<uint8_t*>(t.m) + at, *v = static_cast<uint8_t*>(t.v) + at;
    const bool some = left > 0;
    const bool wide = left >= V && ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g)) & 15) == 0 &&
                      ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 7) == 0;
    float pp[V], gg[V], mm[V], ww[V];
    uint32_t mc[V], vc[V];
    float ms = 0, vs = 0;
    if (some) {
        ms = t.m_scale[at / kBlock];
        vs = t.v_scale[at / kBlock];
    }
    if (wide) {
        load<T, V>(p, pp);
        load<T, V>(g, gg);
        const Pack<uint8_t, V> x = *reinterpret_cast<Pack<uint8_t, V>*>(m), y = *reinterpret_cast<Pack<uint8_t, V>*>(v);
#pragma unroll
        for (int e = 0; e < V; ++e) mc[e] = x.e[e], vc[e] = y.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const bool in = e < left;
            pp[e] = in ? widen<T>(p[e]) : 0.0f;
            gg[e] = in ? widen<T>(g[e]) : 0.0f;
            mc[e] = in ? m[e] : 0;
            vc[e] = in ? v[e] : 0;
        }
    }
    uint32_t mtop = 0, wtop = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        mm[e] = Code<false>::value(mc[e], ms);
        const float w = Code<true>::value(vc[e], vs);
        float vv = w * w;
        pp[e] = updated(pp[e], grad_scale ? gg[e] * gs : gg[e], mm[e], vv, ww[e], f);
        const bool in = wide || e < left;
        if (!in) mm[e] = ww[e] = 0;
        mtop = max(mtop, magnitude(mm[e]));
        wtop = max(wtop, magnitude(ww[e]));
    }
    mtop = max_of_16(mtop);
    wtop = max_of_16(wtop);
    ms = __uint_as_float(max(mtop, uint32_t(__shfl_xor(int(mtop), 16)))) * float(1 / 1.9375);
    vs = __uint_as_float(max(wtop, uint32_t(__shfl_xor(int(wtop), 16)))) * float(1 / 1.9375);
    if (!some) return;
    Pack<uint8_t, V> x, y;
    const uint64_t key = kDraw ? keys.of[i] : 0;
    const auto codes = [&](auto near) {
        const float mi = near ? 1.0f / ms : 0, vi = near ? 1.0f / vs : 0;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float rm = 0, rv = 0;
            if constexpr (kDraw) drawn(key, at + e, rm, rv);
            x.e[e] = Code<false>::template code<near, kDraw>(mm[e], ms, mi, rm, ms * 0x1p-10f <= ww[e] * 4.0f);
            y.e[e] = Code<true>::template code<near, kDraw>(ww[e], vs, vi, rv, true);
        }
    };
    if (min(ms, vs) >= 0x1p-70f && max(ms, vs) <= 0x1p100f) codes(std::true_type{});
    else codes(std::false_type{});
    if (wide) {
        store<T, V>(p, pp);
        *reinterpret_cast<Pack<uint8_t, V>*>(m) = x;
        *reinterpret_cast<Pack<uint8_t, V>*>(v) = y;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (e < left) {
                p[e] = narrow<T>(pp[e]);
                m[e] = x.e[e];
                v[e] = y.e[e];
            }
        }
    }
    if (threadIdx.x % 32 == 0) {
        t.m_scale[at / kBlock] = ms;
        t.v_scale[at / kBlock] = vs;
    }
}

__global__ __launch_bounds__(kThreads) void k_adamw_read(Tensors a) {
#pragma clang fp contract(off)
    constexpr int V = 4, kShare = kThreads * V;
    const int i = owner(a, blockIdx.x);
    const fcqt_adamw_tensor& t = a.t[i];
    const int64_t at = int64_t(blockIdx.x - a.first[i]) * kShare + threadIdx.x * V;
    const int64_t left = t.n - at;
    if (left <= 0) return;
    float *om = static_cast<float*>(t.p) + at, *ov = static_cast<float*>(const_cast<void*>(t.g)) + at;
    const uint8_t *m = static_cast<const uint8_t*>(t.m) + at, *v = static_cast<const uint8_t*>(t.v) + at;
    const float ms = t.m_scale[at / kBlock], vs = t.v_scale[at / kBlock];
    const bool wide = left >= V && ((reinterpret_cast<uintptr_t>(om) | reinterpret_cast<uintptr_t>(ov)) & 15) == 0 &&
                      ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 3) == 0;
    if (wide) {
        const Pack<uint8_t, V> x = *reinterpret_cast<const Pack<uint8_t, V>*>(m), y = *reinterpret_cast<const Pack<uint8_t, V>*>(v);
        float mm[V], vv[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            mm[e] = Code<false>::value(x.e[e], ms);
            const float w = Code<true>::value(y.e[e], vs);
            vv[e] = w * w;
        }
        store<float, V>(om, mm);
        store<float, V>(ov, vv);
        return;
    }
    for (int e = 0; e < min(int64_t(V), left); ++e) {
        om[e] = Code<false>::value(m[e], ms);
        const float w = Code<true>::value(v[e], vs);
        ov[e] = w * w;
    }
}

// Launches of at most kMost descriptors and kGrid workgroups (a grid holds less than 2^32 threads): a tensor past that
// goes in pieces of whole blocks. elem, moment: bytes of an element of p and g, of m and v.
constexpr int64_t kGrid = int64_t(1) << 23;

struct Place {
    int64_t tensor, first;
};

template <class Launch>
int in_groups(const fcqt_adamw_tensor* tensors, int64_t count, int64_t share, int elem, int moment, Launch launch) {
    int64_t at = 0, done = 0;                              // the next tensor, and how much of it has been given out
    while (at < count) {
        Tensors a;
        Place begun[kMost];                                // which tensor each descriptor is of, and from where
        a.count = 0;
        int64_t blocks = 0;
        while (at < count && a.count < kMost && blocks < kGrid) {
            const fcqt_adamw_tensor& t = tensors[at];
            const int64_t n = std::min(t.n - done, (kGrid - blocks) * share);
            if (n > 0) {
                const auto moved = [&](const void* p, int64_t bytes) {
                    return p ? static_cast<char*>(const_cast<void*>(p)) + done * bytes : nullptr;
                };
                const auto scale = [&](float* p) { return p ? p + done / kBlock : nullptr; };
                begun[a.count] = {at, done};
                a.t[a.count] = {moved(t.p, elem), moved(t.g, elem), moved(t.m, moment), moved(t.v, moment),
                                scale(t.m_scale), scale(t.v_scale), n};
                a.first[a.count++] = uint32_t(blocks);
                blocks += (n + share - 1) / share;
                done += n;
            }
            if (done >= t.n) ++at, done = 0;
        }
        if (!a.count) break;
        launch(a, dim3(uint32_t(blocks)), begun);
        if (int e = launched()) return e;
    }
    return FCQT_OK;
}

int checked(const fcqt_adamw_tensor* tensors, int64_t count, int elem, int moment, bool scales) {
    if (count < 0 || (count && !tensors)) return FCQT_EARG;
    for (int64_t i = 0; i < count; ++i) {
        const fcqt_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > (int64_t(1) << 40)) return FCQT_EARG;
        if (t.n == 0) continue;
        if (!t.p || !t.g || !t.m || !t.v || (scales && (!t.m_scale || !t.v_scale))) return FCQT_EARG;
        if (!aligned(t.p, elem) || !aligned(t.g, elem) || !aligned(t.m, moment) || !aligned(t.v, moment)) return FCQT_EALIGN;
        if (scales && (!aligned(t.m_scale, 4) || !aligned(t.v_scale, 4))) return FCQT_EALIGN;
    }
    return FCQT_OK;
}

template <class T, bool kDraw>
void launch8(const Tensors& a, dim3 grid, const fcqt_adamw_factors& f, const float* grad_scale, const Keys<kDraw>& keys, hipStream_t stream) {
    k_adamw8<T, kDraw><<<grid, kThreads, 0, stream>>>(a, f, grad_scale, keys);
}

template <bool kDraw>
void launch8(const Tensors& a, dim3 grid, int32_t dtype, const fcqt_adamw_factors& f, const float* grad_scale, const Keys<kDraw>& keys,
             hipStream_t stream) {
    if (dtype == FCQT_F32) launch8<float>(a, grid, f, grad_scale, keys, stream);
    else if (dtype == FCQT_BF16) launch8<bf16>(a, grid, f, grad_scale, keys, stream);
    else launch8<f16>(a, grid, f, grad_scale, keys, stream);
}

}  // namespace

extern "C" int fcqt_adamw(const fcqt_adamw_tensor* tensors, int64_t count, int32_t dtype, int32_t bits,
                          const fcqt_adamw_factors* factors, const float* grad_scale, hipStream_t stream) {
    if (!factors || !known(dtype) || (bits != 8 && bits != 32)) return FCQT_EARG;
    if (int e = checked(tensors, count, size_of(dtype), bits / 8, bits == 8)) return e;
    if (!aligned(grad_scale, 4)) return FCQT_EALIGN;
    const fcqt_adamw_factors f = *factors;
    return in_groups(tensors, count, bits == 32 ? kThreads * 4 : kThreads * 8, size_of(dtype), bits / 8, [&](const Tensors& a, dim3 grid, const Place*) {
        if (bits == 8) return launch8<false>(a, grid, dtype, f, grad_scale, Keys<false>{}, stream);
        if (dtype == FCQT_F32) k_adamw<float><<<grid, kThreads, 0, stream>>>(a, f, grad_scale);
        else if (dtype == FCQT_BF16) k_adamw<bf16><<<grid, kThreads, 0, stream>>>(a, f, grad_scale);
        else k_adamw<f16><<<grid, kThreads, 0, stream>>>(a, f, grad_scale);
    });
}

extern "C" int fcqt_adamw_drawn(const fcqt_adamw_tensor* tensors, int64_t count, int32_t dtype,
                                const fcqt_adamw_factors* factors, const float* grad_scale, uint64_t seed, int64_t step,
                                hipStream_t stream) {
    if (!factors || !known(dtype)) return FCQT_EARG;
    if (int e = checked(tensors, count, size_of(dtype), 1, true)) return e;
    if (!aligned(grad_scale, 4)) return FCQT_EALIGN;
    const fcqt_adamw_factors f = *factors;
    const uint64_t from = mixed(seed) + uint64_t(step);
    return in_groups(tensors, count, kThreads * 8, size_of(dtype), 1, [&](const Tensors& a, dim3 grid, const Place* begun) {
        Keys<true> keys;
        for (int i = 0; i < kMost; ++i)
            keys.of[i] = i >= a.count ? 0 : mixed(from + uint64_t(begun[i].tensor + 1) * 0x9E3779B97F4A7C15ull + uint64_t(begun[i].first) * 0xBB67AE8584CAA73Bull);
        launch8<true>(a, grid, dtype, f, grad_scale, keys, stream);
    });
}

extern "C" int fcqt_adamw_read(const fcqt_adamw_tensor* tensors, int64_t count, hipStream_t stream) {
    if (int e = checked(tensors, count, 4, 1, true)) return e;
    return in_groups(tensors, count, kThreads * 4, 4, 1, [&](const Tensors& a, dim3 grid, const Place*) {
        k_adamw_read<<<grid, kThreads, 0, stream>>>(a);
    });
}
