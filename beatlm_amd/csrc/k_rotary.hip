// Rotary positions of one to three axes (include/beatlm_ops.h).
//
// A thread owns VEC pairs of one row (or VEC channels of the copied tail) and
// walks heads with them: it makes its VEC sines and cosines once, from the
// table's 64-bit revolutions per position (pos * turns, its fraction taken in
// 64 bits: within |pos| 2^-54 revolutions, which is 2^-8 of f32's step at
// positions of 2 million and four steps at 2^31; then one rounding to f32 and a
// sine good to a few steps of 1), and every head of q and k then costs two
// 16-byte loads, six products a pair and two stores. The bound is HBM: each channel in once, out once.
// 32768 rows of 16 + 4 heads of 128, bf16: 74 us, 4.5 TB/s.
#include "ops_device.hpp"

namespace bl {

namespace {

struct RotaryGeometry {
    uint32_t units;        // pair chunks and tail chunks of a head
    uint32_t pair_units;
    uint32_t head_groups;  // threads that share a row's heads
    uint32_t rows;         // rows a workgroup holds at once
    uint32_t first;        // the launch's first row
};

template <typename T, int VEC>
__device__ __forceinline__ void turn_heads(const RotaryParams &p, const bl_heads &in, const bl_heads &out, uint32_t heads, bool copy,
                                           uint32_t row, uint32_t unit, uint32_t first, const RotaryGeometry &geo, const float (&co)[VEC],
                                           const float (&si)[VEC]) {
    const T *src = (const T *)in.data + (uint64_t)row * in.row_stride;
    T *dst = (T *)out.data + (uint64_t)row * out.row_stride;
    if (unit >= geo.pair_units) {  // a chunk of the channels beyond the pairs
        if (!copy) return;
        const uint32_t c = 2 * p.table.pairs + (unit - geo.pair_units) * VEC;
        for (uint32_t h = first; h < heads; h += geo.head_groups) {
            float v[VEC];
            load_vec<T, VEC>(src + (uint64_t)h * in.head_stride + c, v);
            store_vec<T, VEC>(dst + (uint64_t)h * out.head_stride + c, v);
        }
        return;
    }
    const bool halves = p.table.layout == BL_ROTARY_HALVES;
    // Halves: the chunk's first members and its second members lie apart;
    // neighbours: its 2 VEC channels lie in a row.
    const uint32_t c0 = halves ? unit * VEC : unit * 2 * VEC;
    const uint32_t c1 = halves ? c0 + p.table.pairs : c0 + VEC;
    for (uint32_t h = first; h < heads; h += geo.head_groups) {
        float a[VEC], b[VEC];
        load_vec<T, VEC>(src + (uint64_t)h * in.head_stride + c0, a);
        load_vec<T, VEC>(src + (uint64_t)h * in.head_stride + c1, b);
        float u[VEC], w[VEC];
        if (halves) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                u[e] = a[e] * co[e] - b[e] * si[e];
                w[e] = a[e] * si[e] + b[e] * co[e];
            }
        } else if constexpr (VEC == 1) {
            u[0] = a[0] * co[0] - b[0] * si[0];
            w[0] = a[0] * si[0] + b[0] * co[0];
        } else {
#pragma unroll
            for (int e = 0; e < VEC / 2; e++) {
                u[2 * e] = a[2 * e] * co[e] - a[2 * e + 1] * si[e];
                u[2 * e + 1] = a[2 * e] * si[e] + a[2 * e + 1] * co[e];
                w[2 * e] = b[2 * e] * co[VEC / 2 + e] - b[2 * e + 1] * si[VEC / 2 + e];
                w[2 * e + 1] = b[2 * e] * si[VEC / 2 + e] + b[2 * e + 1] * co[VEC / 2 + e];
            }
        }
        store_vec<T, VEC>(dst + (uint64_t)h * out.head_stride + c0, u);
        store_vec<T, VEC>(dst + (uint64_t)h * out.head_stride + c1, w);
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryParams p, RotaryGeometry geo) {
    const uint32_t unit = threadIdx.x % geo.units, rest = threadIdx.x / geo.units;
    const uint32_t group = rest % geo.head_groups, slot = rest / geo.head_groups;
    const uint64_t at = geo.first + (uint64_t)blockIdx.x * geo.rows + slot;
    if (slot >= geo.rows || at >= p.rows) return;
    const uint32_t row = (uint32_t)at;
    float co[VEC], si[VEC];
    if (unit < geo.pair_units) {
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const uint32_t pair = unit * VEC + e;
            const double t = (double)p.positions[(uint64_t)row * p.table.axes + p.table.axis[pair]] * p.table.turns[pair];
            sincospif(2.0f * (float)(t - rint(t)), &si[e], &co[e]);
            si[e] *= p.sign;
        }
    }
    turn_heads<T, VEC>(p, p.q_in, p.q_out, p.q_heads, p.copy_q, row, unit, group, geo, co, si);
    turn_heads<T, VEC>(p, p.k_in, p.k_out, p.k_heads, p.copy_k, row, unit, group, geo, co, si);
}

template <typename T, int VEC>
hipError_t launch(const RotaryParams &p, uint32_t compute_units, hipStream_t s) {
    RotaryGeometry g;
    g.pair_units = p.table.pairs / VEC;
    g.units = g.pair_units + (p.head_dim - 2 * p.table.pairs) / VEC;
    // A row's heads are shared among more threads until the grid fills the
    // chip twice (each then makes the row's sines again, which few rows can
    // afford), or each has one head.
    const uint32_t heads = p.q_heads > p.k_heads ? p.q_heads : p.k_heads;
    g.head_groups = 1;
    while (2 * g.head_groups * g.units <= 256 && g.head_groups < heads &&
           p.rows < 2ull * compute_units * (256 / (g.units * g.head_groups)))
        g.head_groups *= 2;
    g.rows = 256 / (g.units * g.head_groups);
    // A grid has fewer than 2^32 threads: more rows than that take more launches.
    const uint64_t most = 1u << 23, groups = ((uint64_t)p.rows + g.rows - 1) / g.rows;
    for (uint64_t done = 0; done < groups; done += most) {
        g.first = (uint32_t)(done * g.rows);
        const uint32_t grid = (uint32_t)(groups - done < most ? groups - done : most);
        if (const hipError_t e = run_kernel(rotary_kernel<T, VEC>, grid, 256, s, p, g); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_rotary(const RotaryParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s) {
    switch (dtype) {
    case BL_F32: return p.vector ? launch<float, 4>(p, compute_units, s) : launch<float, 1>(p, compute_units, s);
    case BL_F16: return p.vector ? launch<_Float16, 8>(p, compute_units, s) : launch<_Float16, 1>(p, compute_units, s);
    default: return p.vector ? launch<__bf16, 8>(p, compute_units, s) : launch<__bf16, 1>(p, compute_units, s);
    }
}

}  // namespace bl
