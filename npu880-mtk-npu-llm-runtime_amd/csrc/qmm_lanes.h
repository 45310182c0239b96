// qmm_lanes.h — sums and maxima over lanes in the vector registers' own network; loads and stores past the caches.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace qmm {

template <int CTRL> __device__ inline uint32_t lane_moved(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 15, 15, true));
}
template <int CTRL> __device__ inline float lane_moved(float v) { return __uint_as_float(lane_moved<CTRL>(__float_as_uint(v))); }

// f over groups of N neighbouring lanes (16, 32 or 64): every lane gets the result
template <int N, typename F> __device__ inline uint32_t over_lanes(uint32_t v, F f) {
    v = f(v, lane_moved<0xB1>(v));
    v = f(v, lane_moved<0x4E>(v));
    v = f(v, lane_moved<0x141>(v));
    v = f(v, lane_moved<0x140>(v));
    if constexpr (N >= 32) {
        auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(a[0], a[1]);
    }
    if constexpr (N == 64) {
        auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(a[0], a[1]);
    }
    return v;
}
template <int N> __device__ inline float lanes_sum(float v) {
    return __uint_as_float(over_lanes<N>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
template <int N> __device__ inline uint32_t lanes_max(uint32_t v) {
    return over_lanes<N>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int N> __device__ inline float lanes_max(float v) {
    return __uint_as_float(over_lanes<N>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}

// The sum over the lanes that have this lane's number modulo CL (4, 8 or 16).
template <int CL> __device__ inline float columns_sum(float v) {
    if constexpr (CL <= 4) v += lane_moved<0x124>(v);  // turned by 4 of 16, then by 8
    if constexpr (CL <= 8) v += lane_moved<0x128>(v);
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 1 / sqrt(x) to one step of fp32; the instruction takes no number below 2^-126
__device__ inline float inv_root(float x) {
    const bool tiny = x < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? x * 0x1p100f : x) * (tiny ? 0x1p50f : 1.0f);
}
// y / (1 + exp(-y)); 0 where the exponential is past fp32
__device__ inline float silu(float y) {
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f));
}

// Loads and stores that leave the caches to others: of large tensors that are used again only after as much else has passed
typedef float Four __attribute__((ext_vector_type(4)));
template <typename T> __device__ inline T load_past(const T *p) {
    static_assert(sizeof(T) == sizeof(Four));
    return __builtin_bit_cast(T, __builtin_nontemporal_load(reinterpret_cast<const Four *>(p)));
}
template <typename T> __device__ inline void store_past(T *p, T x) {
    static_assert(sizeof(T) == sizeof(Four));
    __builtin_nontemporal_store(__builtin_bit_cast(Four, x), reinterpret_cast<Four *>(p));
}

}  // namespace qmm
