// The plan of a packed attention call (include/beatlm_ops.h): what its
// workspace holds and into how many splits the forward cuts the keys, from
// the sizes alone, so a workspace made for them fits every call.
#include "ops.hpp"

namespace bl {

namespace {
uint64_t rounded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }
}  // namespace

PackedPlan plan_packed(const bl_packed_attention_args &a, uint32_t compute_units) {
    PackedPlan plan{};
    plan.tile_dim = a.head_dim <= 64 ? 64 : 128;
    const uint64_t group = a.q_heads / a.kv_heads;
    // Workgroups of the forward without splits: 128 (row, head) places each.
    const uint64_t whole = (a.q_rows * group / 128 + a.documents) * a.kv_heads;
    const uint32_t keys = a.max_keys && a.max_keys < a.k_rows ? a.max_keys : a.k_rows;
    // Few rows over many keys: the keys are split until the chip has four
    // workgroups a compute unit, each with 256 keys or more.
    const uint64_t wanted = whole ? 4ull * compute_units / whole : 1, most = (keys + 255) / 256;
    plan.splits = (uint32_t)(wanted < most ? wanted : most);
    if (plan.splits < 1) plan.splits = 1;
    const uint64_t places = (uint64_t)a.q_rows * a.q_heads;
    if (plan.splits > 1) {
        plan.partial_bytes = rounded(plan.splits * places * plan.tile_dim * sizeof(float));
        plan.stats_bytes = rounded(plan.splits * places * 2 * sizeof(float));
    }
    plan.forward_bytes = plan.partial_bytes + plan.stats_bytes;
    plan.row_bytes = rounded(places * sizeof(float));
    plan.backward_bytes = 3 * plan.row_bytes;
    return plan;
}

hipError_t launch_packed_forward(const PackedParams &q, const PackedPlan &plan, hipStream_t s) {
    PackedParams p = q;
    p.splits = plan.splits;
    p.partial = (float *)p.a.workspace;
    p.stats = (float *)((char *)p.a.workspace + plan.partial_bytes);
    switch (p.a.dtype) {
    case BL_F32: return packed_forward<float>(p, plan, s);
    case BL_F16: return packed_forward<_Float16>(p, plan, s);
    default: return packed_forward<__bf16>(p, plan, s);
    }
}

hipError_t launch_packed_backward(const PackedParams &q, const PackedPlan &plan, hipStream_t s) {
    PackedParams p = q;
    char *at = (char *)p.a.workspace;
    p.splits = 1;
    p.delta = (float *)at;
    p.largest = (float *)(at + plan.row_bytes);
    p.d_slope = p.g.d_slopes ? (float *)(at + 2 * plan.row_bytes) : nullptr;
    switch (p.a.dtype) {
    case BL_F32: return packed_backward<float>(p, plan, s);
    case BL_F16: return packed_backward<_Float16>(p, plan, s);
    default: return packed_backward<__bf16>(p, plan, s);
    }
}

}  // namespace bl
