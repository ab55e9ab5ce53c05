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
    plan.waves = 4;
    plan.tile_dim = a.head_dim <= 64 ? 64 : 128;
    const uint64_t group = a.q_heads / a.kv_heads, places = (uint64_t)a.q_rows * a.q_heads;
    const uint64_t average = ((uint64_t)a.q_rows * group + a.documents - 1) / a.documents;
    const uint64_t table = (uint64_t)a.cache.max_pages * a.cache.page_rows;
    uint64_t keys = a.max_keys && a.max_keys < table ? a.max_keys : table;
    if (a.window && (uint64_t)a.window + a.q_rows < keys) keys = (uint64_t)a.window + a.q_rows;
    // 16 or 32 places a workgroup, whose waves share its keys, or 128, which share a
    // tile of them. Over long caches two workgroups of 32 keep more loads under way
    // (9 documents of 40 places over 3450 to 11500 keys, heads of 64, f16: 27 us, 128
    // places 35; in codes 31 and 39); over 2049 keys they take 17 us and 16, and 96
    // places 27 and 20.
    plan.blocks = average <= 16 ? 1 : average <= 32 || (average <= 64 && keys >= 4096) ? 2 : PAGED_CHUNK_BLOCKS;
    // Workgroups without splits, and a last, partial one a document.
    const uint64_t whole = ((uint64_t)a.q_rows * group / (16 * plan.blocks) + a.documents) * a.kv_heads, units = compute_units;
    if (plan.blocks == PAGED_CHUNK_BLOCKS) {
        // Equal shares of keys, so that the chip is filled three times over by what
        // the host knows of the lengths: 8 documents, four of 1024 queries over 1641
        // to 6837 keys (544 workgroups), capped, bf16: 264 us, unsplit 300; but four
        // of equal length 380 and 348. Small shares cost more sums than they fill
        // compute units: 300 queries of three documents over 600 keys 31 us in shares
        // of 256, 39 in 128; 100 of one over 2000 24 and 21.
        uint64_t share = keys;
        if (whole < 4 * units) share = (whole * keys + 3 * units - 1) / (3 * units);
        const uint64_t step = share >= 512 ? 512 : whole <= units / 4 ? 128 : 256;
        plan.share = (uint32_t)((share + step - 1) / step * step);
        if (plan.share < step) plan.share = (uint32_t)step;
        plan.splits = (uint32_t)((keys + plan.share - 1) / plan.share);
    } else {
        // Even shares of each document: four workgroups a compute unit (16 tokens over
        // 3449 to 16326 keys, 4 key heads of 128, bf16: 72 us; in two 74, three 72, eight
        // 73; heads of 64 34, 38, 36 and 37. 32 over 3300 to 16153 in codes, 8 key heads
        // of 64: 57; 73, 60 and 62). Heads of 128 in codes are the exception, as a
        // compute unit holds three of their workgroups: 109, and 116, 96 and 104.
        const uint64_t wanted = whole < 4 * units ? (4 * units + whole - 1) / whole : 1, most = (keys + 127) / 128;
        plan.splits = (uint32_t)(wanted < most ? wanted : most);
        // Few keys: eight waves a workgroup, one or two steps each, and no second launch
        // to join splits (one token, 12 heads of 64: over 300 keys 6.8 us, split 9.3;
        // over 700 9.2 and 10.0, over 1500 13.0 and 9.4; heads of 128 8.5 and 10.0, 12.1
        // and 10.4, 18.8 and 11.1).
        if (plan.blocks == 1 && keys <= 512 && whole <= units) plan.waves = 8, plan.splits = 1;
    }
    if (plan.splits < 1) plan.splits = 1;
    if (plan.splits > 1) {
        plan.partial_bytes = rounded(plan.splits * places * plan.tile_dim * sizeof(float));
        plan.stats_bytes = rounded(plan.splits * places * 4 * sizeof(float));
    }
    return plan;
}

hipError_t launch_paged(const bl_paged_attention_args &a, const PagedPlan &plan, hipStream_t s) {
    PagedParams p{};
    p.a = a;
    p.share = plan.share;
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
