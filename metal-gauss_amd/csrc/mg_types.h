// Element types of the token operators (layer norm, rotary positions,
// attention): float32, bfloat16 and float16, computed in float32. Internal
// header.
#pragma once

#include "mg_common.h"

namespace mg {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline bool type_known(int32_t code) { return code == MG_F32 || code == MG_BF16 || code == MG_F16; }

// A launch counts its threads in 32 bits.
inline bool grid_fits(int64_t groups, int threads) {
    return groups * threads < (int64_t(1) << 32);
}

// Elements of one 16-byte access.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// V neighbouring elements from any address an element may have: gfx950 takes
// 16-byte accesses at element alignment, so rows of odd widths and strides
// keep the wide form.
template <typename T, int V, bool kNt = false>
__device__ __forceinline__ void load_vec(const T *p, float (&f)[V]) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    if constexpr (kNt) {
        const vec t = __builtin_nontemporal_load(reinterpret_cast<const vec *>(p));
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)t[i];
    } else {
        T t[V];
        __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)t[i];
    }
}

template <typename T, int V, bool kNt = false>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[V]) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    vec t;
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = (T)f[i];
    if constexpr (kNt) {
        __builtin_nontemporal_store(t, reinterpret_cast<vec *>(p));
    } else {
        __builtin_memcpy(p, &t, sizeof(t));
    }
}

// The same at element `at` of a row of n: what lies past the row reads as 0
// and is not written.
template <typename T, int V, bool kNt = false>
__device__ __forceinline__ void load_row(const T *row, int at, int n, float (&f)[V]) {
    if (at + V <= n) {
        load_vec<T, V, kNt>(row + at, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = at + i < n ? (float)row[at + i] : 0.f;
    }
}

template <typename T, int V, bool kNt = false>
__device__ __forceinline__ void store_row(T *row, int at, int n, const float (&f)[V]) {
    if (at + V <= n) {
        store_vec<T, V, kNt>(row + at, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i < n) row[at + i] = (T)f[i];
    }
}

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum_all(float v) {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_sum_to_lane63(v)), 63));
}

}  // namespace mg
