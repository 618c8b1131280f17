// What the sequence operators' kernels share: element types, wide loads and stores, reductions over lane groups.
#pragma once

#include <cstdint>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/flashcqt_seq.h"

namespace fcqt_seq {

int note(hipError_t e);                                   // keeps the error's text; FCQT_OK or FCQT_ELAUNCH

inline int launched() { return note(hipGetLastError()); }

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int size_of(int32_t dtype) { return dtype == FCQT_F32 ? 4 : 2; }

inline bool known(int32_t dtype) { return dtype == FCQT_F32 || dtype == FCQT_BF16 || dtype == FCQT_F16; }

struct bf16 {
    uint16_t bits;
};
struct f16 {
    uint16_t bits;
};

template <class T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen(float x) { return x; }
template <>
__device__ __forceinline__ float widen(bf16 x) { return __uint_as_float(uint32_t(x.bits) << 16); }
template <>
__device__ __forceinline__ float widen(f16 x) { return float(__builtin_bit_cast(_Float16, x.bits)); }

// to the nearest, ties to even
template <class T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow(float x) { return x; }
template <>
__device__ __forceinline__ bf16 narrow(float x) { return {__builtin_bit_cast(uint16_t, static_cast<__bf16>(x))}; }
template <>
__device__ __forceinline__ f16 narrow(float x) { return {__builtin_bit_cast(uint16_t, static_cast<_Float16>(x))}; }

// V consecutive elements as one load or store
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
    T e[V];
};

template <class T, int V>
__device__ __forceinline__ void load(const T* p, float (&x)[V]) {
    const Pack<T, V> a = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = widen<T>(a.e[i]);
}

template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&x)[V]) {
    Pack<T, V> a;
#pragma unroll
    for (int i = 0; i < V; ++i) a.e[i] = narrow<T>(x[i]);
    *reinterpret_cast<Pack<T, V>*>(p) = a;
}

// rotation of a lane's value inside its row of 16 lanes
template <int kBy>
__device__ __forceinline__ float row_ror(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + kBy, 0xf, 0xf, false));
}

__device__ __forceinline__ float sum_of_16(float x) {
    x += row_ror<8>(x);
    x += row_ror<4>(x);
    x += row_ror<2>(x);
    return x + row_ror<1>(x);
}

// the largest magnitude, as bits: their order is that of the magnitudes, and a NaN is above all of them
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t max_of_16(uint32_t x) {
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x128, 0xf, 0xf, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x124, 0xf, 0xf, false)));
    x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x122, 0xf, 0xf, false)));
    return max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x121, 0xf, 0xf, false)));
}

}  // namespace fcqt_seq
