// paged_types.hpp -- vector loads and stores of fp32, bf16 and f16 runs with
// fp32 values in registers (rounded to nearest even on the way out).
#pragma once

#include "common.hpp"

namespace gfh {

// N consecutive elements, aligned to min(16, N * sizeof(T)) bytes.
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T *p, float (&x)[N]) {
    constexpr int kPer = N * sizeof(T) <= 16 ? N : 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kPer)));
    typedef float fvec __attribute__((ext_vector_type(kPer)));
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
        const fvec v = __builtin_convertvector(reinterpret_cast<const vec *>(p)[i], fvec);
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[i * kPer + e] = v[e];
    }
}
// ONCE: nothing else touches them (nontemporal).
template <int N, bool ONCE = false, typename T>
__device__ __forceinline__ void store_vec(T *p, const float (&x)[N]) {
    constexpr int kPer = N * sizeof(T) <= 16 ? N : 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kPer)));
    typedef float fvec __attribute__((ext_vector_type(kPer)));
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
        fvec v;
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[e] = x[i * kPer + e];
        vec *const at = reinterpret_cast<vec *>(p) + i;
        if constexpr (ONCE)
            __builtin_nontemporal_store(__builtin_convertvector(v, vec), at);
        else
            *at = __builtin_convertvector(v, vec);
    }
}

}  // namespace gfh
