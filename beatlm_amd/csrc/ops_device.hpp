// What the packed sublayer's kernels share: their launch, 16-byte chunks of the
// three element types as f32 values, and their rounding back (to nearest even,
// once, at the store).
#pragma once

#include "device_common.hpp"
#include "ops.hpp"

namespace bl {

// Launches a kernel and returns that launch's own status: the thread's last
// error may be the host's, from before the call.
template <typename... P>
hipError_t run_kernel(void (*kernel)(P...), dim3 grid, uint32_t threads, hipStream_t s, const P &...params) {
    void *args[] = {(void *)&params...};
    return hipLaunchKernel((const void *)kernel, grid, dim3(threads), args, 0, s);
}

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
