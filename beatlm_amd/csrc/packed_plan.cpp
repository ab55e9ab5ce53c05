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
    const uint64_t group = a.q_heads / a.kv_heads, places = (uint64_t)a.q_rows * a.q_heads, key_places = (uint64_t)a.k_rows * a.kv_heads;
    const uint32_t keys = a.max_keys && a.max_keys < a.k_rows ? a.max_keys : a.k_rows;
    // Workgroups without splits: 128 (row, head) places or 128 keys each, and
    // a last, partial one a document.
    const uint64_t rows_whole = (a.q_rows * group / ROWS + a.documents) * a.kv_heads;
    const uint64_t keys_whole = ((uint64_t)a.k_rows / ROWS + a.documents) * a.kv_heads;
    // The streamed side is split where there are few workgroups, each split
    // keeping 64 streamed rows or more. The forward splits where the chip is
    // not covered once, then to four workgroups a compute unit (16 tokens over
    // 3449 to 16326 keys 71 us, two 83; packed images that cover it, 360 workgroups: 49
    // us unsplit, 63 in three). Decoding steps crosses the same line, though its
    // sums are few: of ragged caches of 1724 to 8163 keys, 32 heads of 128 over 8,
    // bf16, 31 (248 workgroups, in four) take 131 us, 32 (256, unsplit) 181; of
    // caches of 8192 each, 193 and 197. The backward's causal rows are longer and its
    // workgroups larger: it splits to two a unit (8192 tokens, 260 workgroups:
    // d_k and d_v 0.81 ms in two, 1.3 unsplit; six texts, 468 workgroups, forward
    // and backward 112 us unsplit, 135 with the three a unit that split them).
    const uint64_t units = compute_units;
    const auto splits = [&](uint64_t wanted, uint64_t streamed) {
        const uint64_t most = (streamed + 63) / 64, n = wanted < most ? wanted : most;
        return (uint32_t)(n < 1 ? 1 : n > 1024 ? 1024 : n);
    };
    const auto twice = [&](uint64_t whole) { return whole ? (2 * units + whole / 2) / whole : 1; };
    // Documents of few places, 32 on average at most: workgroups of 32, where
    // there is a kernel for them (heads of up to 64 in f32).
    plan.few = a.dtype == BL_F32 && plan.tile_dim == 64 && (uint64_t)a.q_rows * group <= (uint64_t)FEW_ROWS * a.documents;
    const uint64_t forward_whole = plan.few ? ((uint64_t)a.q_rows * group / FEW_ROWS + a.documents) * a.kv_heads : rows_whole;
    plan.splits = splits(forward_whole && forward_whole < units ? (plan.few ? 2 : 4) * units / forward_whole : 1, keys);
    plan.splits_q = splits(twice(rows_whole), keys);
    plan.splits_kv = splits(twice(keys_whole), (uint64_t)a.q_rows * group);
    if (plan.splits > 1) {
        plan.partial_bytes = rounded(plan.splits * places * plan.tile_dim * sizeof(float));
        plan.stats_bytes = rounded(plan.splits * places * 2 * sizeof(float));
    }
    plan.forward_bytes = plan.partial_bytes + plan.stats_bytes;
    plan.row_bytes = rounded(places * sizeof(float));
    const uint64_t of_q = plan.splits_q > 1 ? plan.splits_q * 2 * places * plan.tile_dim * sizeof(float) : 0;
    const uint64_t of_kv = plan.splits_kv > 1 ? plan.splits_kv * 2 * key_places * plan.tile_dim * sizeof(float) : 0;
    plan.back_partial_bytes = rounded(of_q > of_kv ? of_q : of_kv);  // one after the other
    plan.back_stats_bytes = plan.splits_q > 1 ? rounded(plan.splits_q * places * 4 * sizeof(float)) : 0;
    plan.norm_bytes = a.dtype == BL_F16 ? rounded(keys_whole * sizeof(float)) : 0;
    plan.backward_bytes = 3 * plan.row_bytes + plan.back_partial_bytes + plan.back_stats_bytes + plan.norm_bytes;
    return plan;
}

hipError_t launch_packed_forward(const PackedParams &q, const PackedPlan &plan, hipStream_t s) {
    PackedParams p = q;
    p.splits = plan.splits;
    p.few = plan.few;
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
    p.splits_q = plan.splits_q;
    p.splits_kv = plan.splits_kv;
    p.delta = (float *)at;
    p.bound = (float *)(at + plan.row_bytes);
    p.d_slope = (float *)(at + 2 * plan.row_bytes);
    p.partial = (float *)(at + 3 * plan.row_bytes);
    p.stats = (float *)(at + 3 * plan.row_bytes + plan.back_partial_bytes);
    p.norms = (float *)(at + 3 * plan.row_bytes + plan.back_partial_bytes + plan.back_stats_bytes);
    switch (p.a.dtype) {
    case BL_F32: return packed_backward<float>(p, plan, s);
    case BL_F16: return packed_backward<_Float16>(p, plan, s);
    default: return packed_backward<__bf16>(p, plan, s);
    }
}

}  // namespace bl
