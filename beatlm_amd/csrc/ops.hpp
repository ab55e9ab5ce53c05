// The packed attention sublayer's operators (include/beatlm_ops.h): what the
// host side (ops.cpp, packed_plan.cpp) hands to the kernels (k_norm.hip,
// k_rotary.hip, k_packed.inc). The launch functions check nothing: ops.cpp has.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/beatlm_ops.h"

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

}  // namespace bl
