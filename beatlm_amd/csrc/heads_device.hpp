// What the kernels that work on single heads share (k_heads.hip, k_cache.hip):
// which thread has which channels of which head and row, the sines and cosines
// of a workgroup's rows, and a head's norm and rotation.
//
// A head is `units` chunks: VEC pairs (two accesses of VEC channels), then VEC
// channels of the rest. `lanes` threads have a head, UP units each, so a head's
// sums stay within a wave; they walk the row's heads head_groups at a time. The
// sines and cosines of the workgroup's rows are made once, a thread a pair, and
// lie in LDS.
#pragma once

#include "ops_device.hpp"

namespace bl {

struct HeadsGeometry {
    uint32_t units, pair_units;
    uint32_t lanes;        // a power of two up to 64
    uint32_t head_groups;  // a power of two
    uint32_t rows;         // 256 / (lanes * head_groups): rows a workgroup holds at once
    uint32_t first;        // the launch's first row
    uint32_t span;         // of the backward: a workgroup's rows, a multiple of `rows`
};

// Units of a thread: heads of 256 channels with single elements have 255.
template <int VEC> constexpr int UNITS = VEC == 1 ? 4 : 1;

// The lanes of a head, then heads at once until the rows fill the chip `times`
// over (a workgroup has 256 threads) or each has its own.
inline HeadsGeometry heads_geometry(uint32_t vec, uint32_t pairs, uint32_t head_dim, uint32_t heads, uint32_t rows, uint32_t least_lanes, uint64_t workgroups) {
    HeadsGeometry g{};
    g.pair_units = pairs / vec;
    g.units = g.pair_units + (head_dim - 2 * pairs) / vec;
    const uint32_t up = vec == 1 ? 4 : 1;
    g.lanes = least_lanes;
    while (g.lanes * up < g.units) g.lanes *= 2;
    g.head_groups = 1;
    while (2 * g.head_groups * g.lanes <= 256 && 2 * g.head_groups <= heads && rows < workgroups * (256 / (g.lanes * g.head_groups))) g.head_groups *= 2;
    g.rows = 256 / (g.lanes * g.head_groups);
    return g;
}

struct Seat {
    uint32_t lane, group, slot;
    __device__ __forceinline__ explicit Seat(const HeadsGeometry &g) {
        lane = threadIdx.x % g.lanes;
        const uint32_t rest = threadIdx.x / g.lanes;
        group = rest % g.head_groups;
        slot = rest / g.head_groups;
    }
};

// A unit's channels: VEC from c0 on and, of pairs, VEC from c1 on.
template <int VEC> struct Chunk {
    uint32_t unit, c0, c1;
    bool there, pair;
    Chunk() = default;
    __device__ __forceinline__ Chunk(const HeadsGeometry &g, uint32_t pairs, uint32_t layout, uint32_t u) {
        const bool halves = layout == BL_ROTARY_HALVES;
        unit = u;
        there = u < g.units;
        pair = u < g.pair_units;
        c0 = pair ? (halves ? u * VEC : u * 2 * VEC) : 2 * pairs + (u - g.pair_units) * VEC;
        c1 = halves ? c0 + pairs : c0 + VEC;
    }
};
// A thread's units of a head.
template <int VEC>
__device__ __forceinline__ void chunks_of(const HeadsGeometry &g, const bl_rotary_table &table, uint32_t lane, Chunk<VEC> (&c)[UNITS<VEC>]) {
#pragma unroll
    for (int k = 0; k < UNITS<VEC>; k++) c[k] = Chunk<VEC>(g, table.pairs, table.layout, lane + k * g.lanes);
}

// Sums over a head's lanes (aligned in the wave), in each of them.
__device__ __forceinline__ float lanes_sum(float v, uint32_t lanes) {
    if (lanes > 1) v = dpp_add<0xB1>(v);
    if (lanes > 2) v = dpp_add<0x4E>(v);
    if (lanes > 4) v = dpp_add<0x141>(v);
    if (lanes > 8) v = dpp_add<0x140>(v);
    if (lanes > 16) v = sum_xor16(v);
    if (lanes > 32) v = sum_xor32(v);
    return v;
}
__device__ __forceinline__ double lanes_sum(double v, uint32_t lanes) {
    for (uint32_t o = 1; o < lanes; o *= 2) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

// A thread's channels of a head, first VEC from c0, then VEC from c1; zeros
// where there are none.
template <int VEC, typename F> struct Channels {
    static constexpr int UP = UNITS<VEC>;
    F v[UP][2 * VEC];

    template <typename T>
    __device__ __forceinline__ void load(const T *head, const Chunk<VEC> (&c)[UP]) {
#pragma unroll
        for (int k = 0; k < UP; k++) {
            float a[VEC] = {}, b[VEC] = {};
            if (c[k].there) load_vec<T, VEC>(head + c[k].c0, a);
            if (c[k].pair) load_vec<T, VEC>(head + c[k].c1, b);
#pragma unroll
            for (int e = 0; e < VEC; e++) v[k][e] = a[e], v[k][VEC + e] = b[e];
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T *head, const Chunk<VEC> (&c)[UP]) const {
#pragma unroll
        for (int k = 0; k < UP; k++) {
            float a[VEC], b[VEC];
#pragma unroll
            for (int e = 0; e < VEC; e++) a[e] = (float)v[k][e], b[e] = (float)v[k][VEC + e];
            if (c[k].there) store_vec<T, VEC>(head + c[k].c0, a);
            if (c[k].pair) store_vec<T, VEC>(head + c[k].c1, b);
        }
    }
    __device__ __forceinline__ F sum(uint32_t lanes) const {
        F s = 0;
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) s += v[k][e];
        return lanes_sum(s, lanes);
    }
    __device__ __forceinline__ F dot(const Channels &o, uint32_t lanes) const {
        F s = 0;
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) s += v[k][e] * o.v[k][e];
        return lanes_sum(s, lanes);
    }
    // Less `by`, where there are channels.
    __device__ __forceinline__ void less(F by, const Chunk<VEC> (&c)[UP]) {
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                v[k][e] -= c[k].there ? by : F(0);
                v[k][VEC + e] -= c[k].pair ? by : F(0);
            }
    }
    __device__ __forceinline__ void times(F by) {
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) v[k][e] *= by;
    }
    __device__ __forceinline__ void times(const Channels &o) {
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) v[k][e] *= o.v[k][e];
    }
    // To n, and rstd. A head's mean comes off before its squares are summed.
    __device__ __forceinline__ F normalise(uint32_t norm, float epsilon, uint32_t head_dim, uint32_t lanes, const Chunk<VEC> (&c)[UP]) {
        if (norm == BL_HEAD_NORM_CENTRED) less(sum(lanes) / (F)head_dim, c);
        const F rstd = inverse_root(dot(*this, lanes) / (F)head_dim + (F)epsilon);
        times(rstd);
        return rstd;
    }
};

// What a thread reads of a head, as it lies in memory: the next head's, on its way.
template <typename T, int VEC> struct Raw {
    static constexpr int UP = UNITS<VEC>;
    typedef T V __attribute__((ext_vector_type(VEC)));
    V first[UP], second[UP];
    __device__ __forceinline__ void load(const T *head, const Chunk<VEC> (&c)[UP]) {
#pragma unroll
        for (int k = 0; k < UP; k++) {
            first[k] = second[k] = V{};
            if (c[k].there) first[k] = *(const V *)(head + c[k].c0);
            if (c[k].pair) second[k] = *(const V *)(head + c[k].c1);
        }
    }
    template <typename F> __device__ __forceinline__ void to(Channels<VEC, F> &x) const {
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) x.v[k][e] = (F)(float)first[k][e], x.v[k][VEC + e] = (F)(float)second[k][e];
    }
};

// The weights: ones without any.
template <int VEC, typename F, typename T>
__device__ __forceinline__ Channels<VEC, F> weights_of(const void *gamma, const Chunk<VEC> (&c)[UNITS<VEC>]) {
    Channels<VEC, F> g;
    if (gamma) {
        g.load((const T *)gamma, c);
    } else {
#pragma unroll
        for (int k = 0; k < UNITS<VEC>; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) g.v[k][e] = 1;
    }
    return g;
}

// A thread's cosines and sines.
template <int VEC, typename F> struct Turn {
    static constexpr int UP = UNITS<VEC>;
    F co[UP][VEC], si[UP][VEC];
    template <typename S>
    __device__ __forceinline__ void load(const S *cosines, const S *sines, const Chunk<VEC> (&c)[UP]) {
#pragma unroll
        for (int k = 0; k < UP; k++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                co[k][e] = c[k].pair ? (F)cosines[c[k].unit * VEC + e] : F(1);
                si[k][e] = c[k].pair ? (F)sines[c[k].unit * VEC + e] : F(0);
            }
    }
    // sign -1: back.
    __device__ __forceinline__ void apply(Channels<VEC, F> &x, uint32_t layout, F sign, const Chunk<VEC> (&c)[UP]) const {
#pragma unroll
        for (int k = 0; k < UP; k++) {
            if (!c[k].pair) continue;
            if (layout == BL_ROTARY_HALVES || VEC == 1) {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const F a = x.v[k][e], b = x.v[k][VEC + e], s = sign * si[k][e];
                    x.v[k][e] = a * co[k][e] - b * s;
                    x.v[k][VEC + e] = a * s + b * co[k][e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const F a = x.v[k][2 * e], b = x.v[k][2 * e + 1], s = sign * si[k][e];
                    x.v[k][2 * e] = a * co[k][e] - b * s;
                    x.v[k][2 * e + 1] = a * s + b * co[k][e];
                }
            }
        }
    }
};

// A register that the compiler takes for new: what is loaded by way of it is not
// kept over a loop's turns.
__device__ __forceinline__ uint32_t fresh(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ void sine_of(double t, float &si, float &co) { sincospif(2.0f * (float)t, &si, &co); }
__device__ __forceinline__ void sine_of(double t, double &si, double &co) { sincospi(2.0 * t, &si, &co); }

// A head's rotation and weights from LDS, not kept in registers over the heads.
template <int VEC, typename F, typename S>
__device__ __forceinline__ void turn_by(Channels<VEC, F> &x, const S *cosines, const S *sines, uint32_t layout, F sign, const Chunk<VEC> (&c)[UNITS<VEC>]) {
    Turn<VEC, F> turn;
    const uint32_t at = fresh(0);
    turn.load(cosines + at, sines + at, c);
    turn.apply(x, layout, sign, c);
}
template <int VEC, typename F>
__device__ __forceinline__ void weigh_by(Channels<VEC, F> &x, const float *weights, const Chunk<VEC> (&c)[UNITS<VEC>]) {
    Channels<VEC, F> w;
    w.load(weights + fresh(0), c);
    x.times(w);
}
// Both tensors' weights to LDS, ones without any.
template <typename T, int MOST>
__device__ __forceinline__ void put_weights(const HeadsParams &p, float (&weights)[2][MOST]) {
    for (uint32_t n = threadIdx.x; n < p.head_dim; n += 256) {
        weights[0][n] = p.q_gamma ? (float)((const T *)p.q_gamma)[n] : 1.0f;
        weights[1][n] = p.k_gamma ? (float)((const T *)p.k_gamma)[n] : 1.0f;
    }
}

// The sines and cosines of `rows` rows, the first of them `first`, [rows][pairs];
// position(slot, row, axis) of rows up to `last`. Angles are reduced in 64 bits.
template <typename F, typename Position>
__device__ __forceinline__ void make_sines(const bl_rotary_table &table, uint32_t rows, uint64_t first, uint64_t last, F *cosines, F *sines, Position position) {
    if (table.pairs == 0) return;
    for (uint32_t i = threadIdx.x; i < rows * table.pairs; i += 256) {
        const uint32_t slot = i / table.pairs, pair = i - slot * table.pairs;
        if (first + slot >= last) continue;
        const double t = (double)position(slot, first + slot, table.axis[pair]) * table.turns[pair];
        sine_of(t - rint(t), sines[i], cosines[i]);
    }
}

}  // namespace bl
