// Norms of each head of queries and keys with their rotary positions, and the
// gradients (include/beatlm_cache.h).
//
// A head's channels are in registers from the load to the store (heads_device.hpp):
// its sums are over the few lanes that have it. The bound is HBM: forward each
// channel in once, out once; backward x and dy in, dx out, with the statistics
// made again from x, which costs no byte more. 32768 rows of 16 + 4 heads of 128,
// bf16: forward 69 us, 4.9 TB/s; backward 120 us, 4.2 TB/s, three workgroups a
// compute unit, and 4.4 us for the launch that adds the weights' sums (with
// weights and sines in registers, and no head under way while one is summed, 180).
#include "heads_device.hpp"

namespace bl {

namespace {

template <typename T, int VEC>
__device__ __forceinline__ void forward_heads(const HeadsParams &p, const HeadsGeometry &g, const Seat &seat, uint64_t row, const bl_heads &in, const bl_heads &out,
                                              uint32_t heads, const void *gamma, const Chunk<VEC> (&c)[UNITS<VEC>], const Turn<VEC, float> &turn) {
    if (seat.group >= heads) return;
    const Channels<VEC, float> weights = weights_of<VEC, float, T>(gamma, c);
    const T *src = (const T *)in.data + row * in.row_stride;
    T *dst = (T *)out.data + row * out.row_stride;
    for (uint32_t h = seat.group; h < heads; h += g.head_groups) {
        Channels<VEC, float> x;
        x.load(src + (uint64_t)h * in.head_stride, c);
        x.normalise(p.norm, p.epsilon, p.head_dim, g.lanes, c);
        x.times(weights);
        turn.apply(x, p.table.layout, 1.0f, c);
        x.store(dst + (uint64_t)h * out.head_stride, c);
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void forward_kernel(HeadsParams p, HeadsGeometry g) {
    constexpr int UP = UNITS<VEC>;
    __shared__ __attribute__((aligned(16))) float cosines[256 * UP * VEC], sines[256 * UP * VEC];
    const Seat seat(g);
    const uint64_t first = g.first + (uint64_t)blockIdx.x * g.rows, row = first + seat.slot;
    make_sines(p.table, g.rows, first, p.rows, cosines, sines, [&](uint32_t, uint64_t r, uint32_t axis) { return p.positions[r * p.table.axes + axis]; });
    __syncthreads();
    if (row >= p.rows) return;
    Chunk<VEC> c[UP];
    chunks_of<VEC>(g, p.table, seat.lane, c);
    Turn<VEC, float> turn;
    turn.load(cosines + seat.slot * p.table.pairs, sines + seat.slot * p.table.pairs, c);
    forward_heads<T, VEC>(p, g, seat, row, p.q_in, p.q_out, p.q_heads, p.q_gamma, c, turn);
    forward_heads<T, VEC>(p, g, seat, row, p.k_in, p.k_out, p.k_heads, p.k_gamma, c, turn);
}

// `sines`: LDS, the row's; the weights lie there too, as they were read, and
// neither is kept in registers over the heads: with them a SIMD has room for five
// waves instead of three.
template <typename T, int VEC>
__device__ __forceinline__ void backward_heads(const HeadsParams &p, const HeadsGeometry &g, const Seat &seat, uint64_t row, const bl_heads &in, const bl_heads &d_out,
                                               const bl_heads &d_in, uint32_t heads, const float *weights, const Chunk<VEC> (&c)[UNITS<VEC>],
                                               const float *cosines, const float *sines, Channels<VEC, float> &d_gamma) {
    if (seat.group >= heads) return;
    const T *src = (const T *)in.data + row * in.row_stride, *dy = (const T *)d_out.data + row * d_out.row_stride;
    T *dst = (T *)d_in.data + row * d_in.row_stride;
    const float each = 1.0f / (float)p.head_dim;
    Raw<T, VEC> x, y;
    x.load(src + (uint64_t)seat.group * in.head_stride, c);
    y.load(dy + (uint64_t)seat.group * d_out.head_stride, c);
    for (uint32_t h = seat.group; h < heads; h += g.head_groups) {
        Channels<VEC, float> n, z;
        x.to(n);
        y.to(z);
        if (h + g.head_groups < heads) {  // the next head's on their way
            x.load(src + (uint64_t)(h + g.head_groups) * in.head_stride, c);
            y.load(dy + (uint64_t)(h + g.head_groups) * d_out.head_stride, c);
        }
        const float rstd = n.normalise(p.norm, p.epsilon, p.head_dim, g.lanes, c);
        turn_by<VEC>(z, cosines, sines, p.table.layout, -1.0f, c);
#pragma unroll
        for (int k = 0; k < UNITS<VEC>; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) d_gamma.v[k][e] += z.v[k][e] * n.v[k][e];
        weigh_by<VEC>(z, weights, c);
        const float along = z.dot(n, g.lanes) * each;
        if (p.norm == BL_HEAD_NORM_CENTRED) z.less(z.sum(g.lanes) * each, c);
#pragma unroll
        for (int k = 0; k < UNITS<VEC>; k++)
#pragma unroll
            for (int e = 0; e < 2 * VEC; e++) z.v[k][e] = (z.v[k][e] - n.v[k][e] * along) * rstd;
        z.store(dst + (uint64_t)h * d_in.head_stride, c);
    }
}

// The workgroup's sum of a thread's d_gamma: its seats of a lane added in order.
template <int VEC>
__device__ __forceinline__ void sum_seats(const HeadsGeometry &g, uint32_t pairs, uint32_t layout, const Channels<VEC, float> &d, float *lds, float *out) {
    constexpr int UP = UNITS<VEC>;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UP; k++)
#pragma unroll
        for (int e = 0; e < 2 * VEC; e++) lds[(k * 2 * VEC + e) * 256 + threadIdx.x] = d.v[k][e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < g.lanes * UP * 2 * VEC; i += 256) {
        const uint32_t lane = i % g.lanes, value = i / g.lanes, k = value / (2 * VEC), e = value % (2 * VEC);
        float s = 0.0f;
        for (uint32_t n = lane; n < 256; n += g.lanes) s += lds[value * 256 + n];
        const Chunk<VEC> c(g, pairs, layout, lane + k * g.lanes);
        if (e < VEC ? c.there : c.pair) out[e < VEC ? c.c0 + e : c.c1 + e - VEC] = s;
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void backward_kernel(HeadsParams p, HeadsGeometry g) {
    constexpr int UP = UNITS<VEC>;
    __shared__ __attribute__((aligned(16))) float lds[2][256 * UP * VEC];  // cosines, sines; in the end the weights' sums
    __shared__ __attribute__((aligned(16))) float weights[2][BL_HEAD_NORM_MAX_HEAD_DIM];
    const Seat seat(g);
    Chunk<VEC> c[UP];
    chunks_of<VEC>(g, p.table, seat.lane, c);
    put_weights<T>(p, weights);
    Channels<VEC, float> d_q = {}, d_k = {};
    // The sines of as many rows at once as there is room for.
    const uint32_t room = p.table.pairs ? (256 * UP * VEC / p.table.pairs) / g.rows * g.rows : g.span, batch = min(room, g.span);
    const uint64_t begin = (uint64_t)blockIdx.x * g.span, end = min(begin + g.span, (uint64_t)p.rows);
    for (uint64_t first = begin; first < end; first += batch) {
        __syncthreads();  // the last rows' sines have been read
        make_sines(p.table, batch, first, end, lds[0], lds[1], [&](uint32_t, uint64_t r, uint32_t axis) { return p.positions[r * p.table.axes + axis]; });
        __syncthreads();
        for (uint64_t row = first + seat.slot; row < min(first + batch, end); row += g.rows) {
            const float *const cosines = lds[0] + (uint32_t)(row - first) * p.table.pairs, *const sines = lds[1] + (uint32_t)(row - first) * p.table.pairs;
            backward_heads<T, VEC>(p, g, seat, row, p.q_in, p.dq_out, p.dq_in, p.q_heads, weights[0], c, cosines, sines, d_q);
            backward_heads<T, VEC>(p, g, seat, row, p.k_in, p.dk_out, p.dk_in, p.k_heads, weights[1], c, cosines, sines, d_k);
        }
    }
    float *out = p.partial + (uint64_t)blockIdx.x * 2 * p.head_dim;
    sum_seats<VEC>(g, p.table.pairs, p.table.layout, d_q, lds[0], out);
    sum_seats<VEC>(g, p.table.pairs, p.table.layout, d_k, lds[0], out + p.head_dim);
}

// The workgroups' sums added: 16 channels a workgroup, 64 threads a channel.
__global__ __launch_bounds__(1024) void weights_kernel(HeadsParams p) {
    __shared__ float lds[64][17];
    const uint32_t c = blockIdx.x * 16 + threadIdx.x % 16, part = threadIdx.x / 16, all = 2 * p.head_dim;
    float s = 0.0f;
    if (c < all)
#pragma unroll 8
        for (uint32_t n = part; n < p.groups; n += 64) s += p.partial[(uint64_t)n * all + c];
    lds[part][threadIdx.x % 16] = s;
    __syncthreads();
    if (part || c >= all) return;
#pragma unroll
    for (int n = 1; n < 64; n++) s += lds[n][threadIdx.x];
    if (c < p.head_dim) {
        if (p.d_q_gamma) p.d_q_gamma[c] = s;
    } else if (p.d_k_gamma) {
        p.d_k_gamma[c - p.head_dim] = s;
    }
}

template <typename T, int VEC>
hipError_t forward(const HeadsParams &p, uint32_t compute_units, hipStream_t s) {
    HeadsGeometry g = heads_geometry(VEC, p.table.pairs, p.head_dim, p.q_heads > p.k_heads ? p.q_heads : p.k_heads, p.rows, 1, 2ull * compute_units);
    // A grid has fewer than 2^32 threads: more rows than that take more launches.
    const uint64_t most = 1u << 23, groups = ((uint64_t)p.rows + g.rows - 1) / g.rows;
    for (uint64_t done = 0; done < groups; done += most) {
        g.first = (uint32_t)(done * g.rows);
        const uint32_t grid = (uint32_t)(groups - done < most ? groups - done : most);
        if (const hipError_t e = run_kernel(forward_kernel<T, VEC>, grid, 256, s, p, g); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename T, int VEC>
hipError_t backward(const HeadsParams &q, hipStream_t s) {
    HeadsParams p = q;
    // As many heads at once as leave a workgroup the fewest turns: 32768 rows of 16 +
    // 4 heads go 4 at a time, 4099 of 9 + 3 two.
    HeadsGeometry g = heads_geometry(VEC, p.table.pairs, p.head_dim, 1, p.rows, 1, 0);
    const uint64_t each = ((uint64_t)p.rows + p.groups - 1) / p.groups;
    uint64_t fewest = ~0ull;
    for (uint32_t at_once = 1; at_once * g.lanes <= 256 && at_once < 2 * (p.q_heads > p.k_heads ? p.q_heads : p.k_heads); at_once *= 2) {
        const uint32_t rows = 256 / (g.lanes * at_once);
        const uint64_t turns = ((p.q_heads + at_once - 1) / at_once + (p.k_heads + at_once - 1) / at_once) * ((each + rows - 1) / rows);
        if (turns <= fewest) fewest = turns, g.head_groups = at_once, g.rows = rows;
    }
    g.span = (uint32_t)((each + g.rows - 1) / g.rows * g.rows);
    if (g.span == 0) g.span = g.rows;
    p.groups = p.rows ? (p.rows + g.span - 1) / g.span : 1;
    const hipError_t e = run_kernel(backward_kernel<T, VEC>, p.groups, 256, s, p, g);
    if (e != hipSuccess || (!p.d_q_gamma && !p.d_k_gamma)) return e;
    return run_kernel(weights_kernel, (2 * p.head_dim + 15) / 16, 1024, s, p);
}

}  // namespace

hipError_t launch_heads_forward(const HeadsParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s) {
    switch (dtype) {
    case BL_F32: return p.vec == 4 ? forward<float, 4>(p, compute_units, s) : forward<float, 1>(p, compute_units, s);
    case BL_F16:
        return p.vec == 8 ? forward<_Float16, 8>(p, compute_units, s) : p.vec == 4 ? forward<_Float16, 4>(p, compute_units, s) : forward<_Float16, 1>(p, compute_units, s);
    default:
        return p.vec == 8 ? forward<__bf16, 8>(p, compute_units, s) : p.vec == 4 ? forward<__bf16, 4>(p, compute_units, s) : forward<__bf16, 1>(p, compute_units, s);
    }
}

hipError_t launch_heads_backward(const HeadsParams &p, uint32_t dtype, uint32_t, hipStream_t s) {
    switch (dtype) {
    case BL_F32: return p.vec == 4 ? backward<float, 4>(p, s) : backward<float, 1>(p, s);
    case BL_F16: return p.vec == 8 ? backward<_Float16, 8>(p, s) : p.vec == 4 ? backward<_Float16, 4>(p, s) : backward<_Float16, 1>(p, s);
    default: return p.vec == 8 ? backward<__bf16, 8>(p, s) : p.vec == 4 ? backward<__bf16, 4>(p, s) : backward<__bf16, 1>(p, s);
    }
}

}  // namespace bl
