// The plan of attention over pages (include/beatlm_cache.h): how many places a
// workgroup has, into how many splits the keys are cut and what the workspace
// holds, from the sizes alone, so a workspace made for them fits every call.
#include "ops.hpp"

namespace bl {

namespace {
uint64_t rounded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }
}  // namespace

PagedPlan plan_paged(const bl_paged_attention_args &a, uint32_t compute_units) {
    PagedPlan plan{};
    plan.tile_dim = a.head_dim <= 64 ? 64 : 128;
    const uint64_t group = a.q_heads / a.kv_heads, places = (uint64_t)a.q_rows * a.q_heads;
    const uint64_t average = ((uint64_t)a.q_rows * group + a.documents - 1) / a.documents;
    plan.blocks = average <= 16 ? 1 : average <= 32 ? 2 : 4;
    const uint64_t table = (uint64_t)a.cache.max_pages * a.cache.page_rows;
    uint64_t keys = a.max_keys && a.max_keys < table ? a.max_keys : table;
    if (a.window && (uint64_t)a.window + a.q_rows < keys) keys = (uint64_t)a.window + a.q_rows;
    // Workgroups without splits, and a last, partial one a document.
    const uint64_t whole = ((uint64_t)a.q_rows * group / (16 * plan.blocks) + a.documents) * a.kv_heads;
    const uint64_t wanted = whole < 4ull * compute_units ? (4ull * compute_units + whole - 1) / whole : 1, most = (keys + 127) / 128;
    plan.splits = (uint32_t)(wanted < most ? wanted : most);
    if (plan.splits < 1) plan.splits = 1;
    if (plan.splits > 1) {
        plan.partial_bytes = rounded(plan.splits * places * plan.tile_dim * sizeof(float));
        plan.stats_bytes = rounded(plan.splits * places * 2 * sizeof(float));
    }
    return plan;
}

hipError_t launch_paged(const bl_paged_attention_args &a, const PagedPlan &plan, hipStream_t s) {
    PagedParams p{};
    p.a = a;
    p.splits = plan.splits;
    p.page_magic = (uint32_t)(((1ull << 32) + a.cache.page_rows - 1) / a.cache.page_rows);
    p.partial = (float *)a.workspace;
    p.stats = (float *)((char *)a.workspace + plan.partial_bytes);
    switch (a.dtype) {
    case BL_F32: return paged_attention<float>(p, plan, s);
    case BL_F16: return paged_attention<_Float16>(p, plan, s);
    default: return paged_attention<__bf16>(p, plan, s);
    }
}

}  // namespace bl
