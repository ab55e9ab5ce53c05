// Device helpers the packed sublayer's kernels share: 16-byte chunks of the
// three element types as f32 values, and their rounding back (to nearest even,
// once, at the store).
#pragma once

#include "device_common.hpp"
#include "ops.hpp"

namespace bl {

// VEC elements at p (16-byte aligned when VEC > 1) as f32.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = (float)p[0];
    } else {
        typedef T V __attribute__((ext_vector_type(VEC)));
        const V x = *(const V *)p;
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = (float)x[e];
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = (T)v[0];
    } else {
        typedef T V __attribute__((ext_vector_type(VEC)));
        V x;
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = (T)v[e];
        *(V *)p = x;
    }
}

}  // namespace bl
