// The packed attention sublayer's operators (include/beatlm_ops.h, include/beatlm_cache.h): what the
// host side (ops.cpp, packed_plan.cpp) hands to the kernels (k_norm.hip,
// k_rotary.hip, k_packed.inc), and cache_ops.cpp and paged_plan.cpp to theirs
// (k_heads.hip, k_cache.hip, k_paged.inc). The launch functions check nothing:
// ops.cpp and cache_ops.cpp have.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/beatlm_cache.h"

namespace bl {

// ---- LayerNorm ----

struct NormParams {
    const void *x, *gamma, *beta, *dy;
    void *y, *dx;
    float *mean, *rstd, *d_gamma, *d_beta;
    float *partial;  // [groups][2][cols]: d_gamma's and d_beta's sums of one workgroup's rows
    uint64_t x_stride, y_stride, dy_stride, dx_stride;
    uint32_t rows, cols, groups;
    float epsilon;
};
// Workgroups that walk the rows, up to `each` of 256 threads a compute unit.
// The backward's workspace holds a partial sum of each.
uint32_t norm_groups(uint32_t rows, uint32_t cols, uint32_t compute_units, uint32_t each);
constexpr uint32_t NORM_FORWARD_GROUPS = 8, NORM_BACKWARD_GROUPS = 3;
hipError_t launch_norm_forward(const NormParams &p, uint32_t dtype, hipStream_t s);
hipError_t launch_norm_backward(const NormParams &p, uint32_t dtype, hipStream_t s);

// ---- rotary positions ----

struct RotaryParams {
    bl_rotary_table table;
    const int32_t *positions;
    bl_heads q_in, q_out, k_in, k_out;
    uint32_t rows, q_heads, k_heads, head_dim;
    float sign;       // -1: the inverse
    bool copy_q, copy_k;  // channels beyond the pairs are copied (not when in place)
    bool vector;
};
hipError_t launch_rotary(const RotaryParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s);

// ---- attention over packed documents ----

// (row, head of a group) places, or keys, of a workgroup.
constexpr int ROWS = 128, FEW_ROWS = 32;

struct PackedParams {
    bl_packed_attention_args a;
    bl_packed_attention_grads g;
    // Where the streamed side is split over workgroups, each split's sums,
    // joined by a launch of its own.
    uint32_t splits, splits_q, splits_kv;
    bool few;        // the forward's workgroups have FEW_ROWS places, not ROWS
    float *partial;  // forward [splits][places][tile_dim]; d_q [splits][2][places][tile_dim]; d_k, d_v [splits][2][k_rows * kv_heads][tile_dim]
    float *stats;    // forward [splits][places][2], d_q [splits][places][4]; places = q_rows * q_heads
    // backward, [q_heads][q_rows] each
    float *delta;    // sum_j P_j dP_j of each row
    float *bound;    // a bound of its |dP| (f16)
    float *d_slope;  // its part of d_slopes
    float *norms;    // [kv_heads][slots of 128 keys]: the values' largest squared norm (f16)
};
struct PackedPlan {
    uint32_t splits, splits_q, splits_kv;
    bool few;
    uint32_t tile_dim;  // channels of the kernels' tiles: 64 or 128
    uint64_t partial_bytes, stats_bytes;                     // forward
    uint64_t row_bytes, back_partial_bytes, back_stats_bytes, norm_bytes; // backward
    uint64_t forward_bytes, backward_bytes;
};
PackedPlan plan_packed(const bl_packed_attention_args &a, uint32_t compute_units);
hipError_t launch_packed_forward(const PackedParams &p, const PackedPlan &plan, hipStream_t s);
hipError_t launch_packed_backward(const PackedParams &p, const PackedPlan &plan, hipStream_t s);

// One element type each (k_packed_*.hip).
template <typename T> hipError_t packed_forward(const PackedParams &p, const PackedPlan &plan, hipStream_t s);
template <typename T> hipError_t packed_backward(const PackedParams &p, const PackedPlan &plan, hipStream_t s);

// ---- norms of each head with their rotary positions ----

struct HeadsParams {
    bl_rotary_table table;   // pairs 0: no rotation
    const int32_t *positions;
    const void *q_gamma, *k_gamma;  // null: ones
    bl_heads q_in, q_out, k_in, k_out;
    bl_heads dq_out, dk_out, dq_in, dk_in;
    float *partial;          // [groups][2][head_dim]: the weights' gradients of one workgroup's rows
    float *d_q_gamma, *d_k_gamma;
    uint32_t rows, q_heads, k_heads, head_dim, norm;
    float epsilon;
    uint32_t groups;         // workgroups that walk the rows of the backward
    uint32_t vec;            // elements of an access: 16 bytes, 8 or one element, as everything is aligned
};
constexpr uint32_t HEADS_BACKWARD_GROUPS = 3;  // a compute unit: as many as there is room for with 16-byte accesses of 16-bit types
hipError_t launch_heads_forward(const HeadsParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s);
hipError_t launch_heads_backward(const HeadsParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s);

// ---- the cache of pages ----

struct AppendParams {
    HeadsParams h;           // k_out is not used
    bl_heads v_in;
    bl_paged_cache cache;
    const int32_t *q_offsets;
    uint32_t documents;
};
hipError_t launch_cache_append(const AppendParams &p, uint32_t dtype, uint32_t compute_units, hipStream_t s);
hipError_t launch_cache_read(const bl_cache_read_args &a, uint32_t compute_units, hipStream_t s);

// ---- attention over pages ----

constexpr uint32_t PAGED_CHUNK_BLOCKS = 8;
struct PagedPlan {
    uint32_t blocks;    // of 16 (query, head of a group) places in a workgroup: 1, 2 or PAGED_CHUNK_BLOCKS
    uint32_t waves;     // of a workgroup, 4 or 8: without splits, of few places
    uint32_t share;     // of chunks: keys of a workgroup, from the first that its places see
    uint32_t splits;    // workgroups that share a document's keys; of chunks the longest one's, and the last takes what is left of a longer one
    uint32_t tile_dim;  // channels of the kernels' tiles: 64 or 128
    uint64_t partial_bytes, stats_bytes;
};
struct PagedParams {
    bl_paged_attention_args a;
    uint32_t share, splits;
    uint32_t page_magic;  // ceil(2^32 / page_rows): n / page_rows is the upper half of n times it, up to BL_CACHE_MAX_KEYS
    float *partial;       // [splits][places][tile_dim]; places = q_rows * q_heads
    float *stats;         // [splits][places][4]: maximum, sum, and how many splits the place has
};
PagedPlan plan_paged(const bl_paged_attention_args &a, uint32_t compute_units);
hipError_t launch_paged(const bl_paged_attention_args &a, const PagedPlan &plan, hipStream_t s);
// One element type each (k_paged_*.hip).
template <typename T> hipError_t paged_attention(const PagedParams &p, const PagedPlan &plan, hipStream_t s);

}  // namespace bl
