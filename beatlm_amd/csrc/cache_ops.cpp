// The host side of the norms of heads and of the cache of pages
// (include/beatlm_cache.h): every check of a call's arguments, and the launch on
// the context's stream. Nothing here allocates or waits.
#include "ops.hpp"
#include "ops_checks.hpp"

#include <utility>

using namespace bl::checks;

namespace {

bool finite_epsilon(float e) { return std::isfinite(e) && e >= 0.0f; }

Named heads_named(const bl_heads &h, uint64_t rows, uint64_t heads, uint64_t head_dim, uint64_t size, const char *name) {
    return {bytes_of(h, rows, heads, head_dim, size), name};
}
Named weights_named(const void *p, uint64_t head_dim, uint64_t size, const char *name) { return {bytes_of({(void *)p, 0, 0}, 1, 1, head_dim, size), name}; }
// Bytes next to each other: indices, weights' gradients, a workspace.
Named block_named(const void *p, uint64_t bytes, const char *name) { return {{(uint64_t)p, 0, 1, 0, p && bytes ? 1u : 0u, bytes}, name}; }
Named positions_named(const bl_rotary_table *t, const int32_t *positions, uint64_t rows) {
    return block_named(t ? positions : nullptr, t ? rows * t->axes * 4 : 0, "positions");
}
// A call's outputs beside indices that it reads.
template <size_t N, size_t M>
int check_outputs_apart(bl_ctx *ctx, const char *what, const Named (&written)[N], const Named (&read)[M]) {
    for (const Named &out : written)
        for (const Named &in : read)
            if (int rc = check_apart(ctx, what, out, in)) return rc;
    return BL_OK;
}

// ---- norms of heads ----

int check_head_norm(bl_ctx *ctx, const bl_head_norm_args *a, const char *what) {
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->head_dim == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: heads of no channels", what);
    if (a->head_dim > BL_HEAD_NORM_MAX_HEAD_DIM)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: heads of %u, at most %u", what, a->head_dim, BL_HEAD_NORM_MAX_HEAD_DIM);
    if (a->norm != BL_HEAD_NORM_RMS && a->norm != BL_HEAD_NORM_CENTRED) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: norm %u", what, a->norm);
    if (!finite_epsilon(a->epsilon)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: an epsilon that is negative or not finite", what);
    if (a->q_heads == 0 && a->k_heads == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no heads", what);
    if (a->rows > 0x7fffffffu || a->q_heads > 65535 || a->k_heads > 65535)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u rows of %u and %u heads", what, a->rows, a->q_heads, a->k_heads);
    return BL_OK;
}

int check_turn(bl_ctx *ctx, const bl_rotary_table *t, const int32_t *positions, uint32_t rows, uint32_t head_dim, bool needed, const char *what) {
    if (!t) return BL_OK;
    if (int rc = check_table(ctx, t, head_dim, what)) return rc;
    if (rows && ((needed && !positions) || !aligned(positions, 4)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: positions are null or misaligned", what);
    return BL_OK;
}

int check_weights(bl_ctx *ctx, const void *gamma, uint64_t size, const char *what, const char *name) {
    return gamma && !aligned(gamma, size) ? refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: %s is misaligned", what, name) : BL_OK;
}

// An output beside what is read: the one input it may be, and others that it may not touch.
int check_in_place(bl_ctx *ctx, const char *what, const Named &out, const bl_heads &o, const Named &in, const bl_heads &i) {
    if (in.bytes.rows == 0 || in.bytes.heads == 0 || out.bytes.rows == 0 || out.bytes.heads == 0) return BL_OK;
    if (o.data == i.data && !same_heads(o, i)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is %s with other strides", what, out.name, in.name);
    return o.data == i.data ? BL_OK : check_apart(ctx, what, out, in);
}

// The widest access that every tensor and the table's sections allow.
struct Widest {
    uint64_t size;
    uint32_t vec;
    explicit Widest(uint32_t dtype) : size(element_size(dtype)), vec((uint32_t)(16 / size)) {}
    void narrow(bool (*fits)(const void *, uint64_t, uint64_t, uint64_t, uint64_t), const void *p, uint64_t row, uint64_t head) {
        while (vec > 1 && !fits(p, row, head, vec, size)) vec = vec == 8 ? 4 : 1;
    }
    static bool fits(const void *p, uint64_t row, uint64_t head, uint64_t n, uint64_t size) { return aligned(p, n * size) && row % n == 0 && head % n == 0; }
    void heads(const bl_heads &h, uint32_t count) {
        if (count) narrow(fits, h.data, h.row_stride, h.head_stride);
    }
    void vector(const void *p) {
        if (p) narrow(fits, p, 0, 0);
    }
    void count(uint32_t n) { narrow(fits, nullptr, n, n); }
};

bl::HeadsParams heads_params(const bl_rotary_table *t, const bl_head_norm_args *a) {
    bl::HeadsParams p{};
    if (t) p.table = *t;
    p.positions = a->positions;
    p.q_gamma = a->q_heads ? a->q_gamma : nullptr;  // weights of no heads are not looked at, and may be any address
    p.k_gamma = a->k_heads ? a->k_gamma : nullptr;
    p.q_in = a->q_in;
    p.q_out = a->q_out;
    p.k_in = a->k_in;
    p.k_out = a->k_out;
    p.rows = a->rows;
    p.q_heads = a->q_heads;
    p.k_heads = a->k_heads;
    p.head_dim = a->head_dim;
    p.norm = a->norm;
    p.epsilon = a->epsilon;
    return p;
}

uint32_t heads_groups(bl_ctx *ctx, const bl_head_norm_args *a) {
    const uint64_t most = (uint64_t)bl_compute_units_of(ctx) * bl::HEADS_BACKWARD_GROUPS;
    return (uint32_t)(a->rows < 1 ? 1 : a->rows < most ? a->rows : most);
}
uint64_t heads_workspace(bl_ctx *ctx, const bl_head_norm_args *a) { return (uint64_t)heads_groups(ctx, a) * 2 * a->head_dim * sizeof(float); }

// ---- the cache ----

uint64_t row_bytes(const bl_paged_cache &c, uint32_t dtype, uint32_t head_dim) {
    return c.kind == BL_CACHE_INT4 ? head_dim / 2 + head_dim / 8 : head_dim * element_size(dtype);
}

int check_cache_sizes(bl_ctx *ctx, const bl_paged_cache &c, uint32_t head_dim, const char *what) {
    if (c.kind > BL_CACHE_INT4) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown cache kind %u", what, c.kind);
    const uint32_t step = c.kind == BL_CACHE_INT4 ? BL_CACHE_GROUP : 8;
    if (head_dim == 0 || head_dim % step || head_dim > BL_ATTENTION_MAX_HEAD_DIM)
        return refuse(ctx, head_dim > BL_ATTENTION_MAX_HEAD_DIM ? BL_ERR_TOO_LARGE : BL_ERR_INVALID_ARGUMENT, "%s: heads of %u, not a multiple of %u up to %u", what,
                      head_dim, step, BL_ATTENTION_MAX_HEAD_DIM);
    if (c.page_rows == 0 || c.page_rows % 16 || c.page_rows > BL_CACHE_MAX_PAGE_ROWS)
        return refuse(ctx, c.page_rows > BL_CACHE_MAX_PAGE_ROWS ? BL_ERR_TOO_LARGE : BL_ERR_INVALID_ARGUMENT, "%s: pages of %u rows, not a multiple of 16 up to %u", what,
                      c.page_rows, BL_CACHE_MAX_PAGE_ROWS);
    if (c.max_pages == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a table of no pages", what);
    if ((uint64_t)c.max_pages * c.page_rows > BL_CACHE_MAX_KEYS || c.pages > 0x7fffffffu)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u pages of %u rows a document, %u in all", what, c.max_pages, c.page_rows, c.pages);
    return BL_OK;
}

// The steps of a side of the cache in falling order of size, and whether no two
// of its rows meet: all rows of a step lie within the next larger one.
struct Steps {
    uint64_t step[4], count[4];
    int n = 0;
    void add(uint64_t s, uint64_t c) {
        if (c > 1) step[n] = s, count[n++] = c;
    }
    bool apart(uint64_t width) {
        for (int i = 1; i < n; i++)
            for (int j = i; j > 0 && step[j] < step[j - 1]; j--) std::swap(step[j], step[j - 1]), std::swap(count[j], count[j - 1]);
        wide extent = width;
        for (int i = 0; i < n; i++) {
            if ((wide)step[i] < extent) return false;
            extent += (wide)step[i] * (count[i] - 1);
        }
        return true;
    }
};
Steps steps_of(const bl_paged_cache &c, const bl_pages &p, uint32_t heads) {
    Steps s;
    s.add(p.page_stride, c.pages);
    s.add(p.row_stride, c.page_rows);
    s.add(p.head_stride, heads);
    return s;
}
// Whether a block of bytes meets a row of one of the n smallest steps, the first
// row at 0; steps sorted, rows apart. A step's copies that the block meets are
// neighbours, and of three the middle one lies in it whole.
bool meets(const Steps &s, int n, wide from, wide to, uint64_t width) {
    if (n == 0) return from < (wide)width && to > 0;
    wide extent = width;
    for (int i = 0; i < n - 1; i++) extent += (wide)s.step[i] * (s.count[i] - 1);
    const wide step = s.step[n - 1];
    if (to <= 0) return false;
    const wide first = from < extent ? 0 : (from - extent) / step + 1, end = (to - 1) / step + 1;
    const wide last = (end < (wide)s.count[n - 1] ? end : (wide)s.count[n - 1]) - 1;
    if (last - first >= 2) return true;
    for (wide i = first; i <= last; i++)
        if (meets(s, n - 1, from - i * step, to - i * step, width)) return true;
    return false;
}

// All the bytes of a side from its first to its last.
Bytes extent_of(const bl_paged_cache &c, const bl_pages &p, uint32_t heads, uint64_t width) {
    const uint64_t last = c.pages ? (c.pages - 1) * p.page_stride + (c.page_rows - 1) * p.row_stride + (heads - 1) * p.head_stride + width : 0;
    return {(uint64_t)p.data, 0, 1, 0, last ? 1u : 0u, last};
}

int check_cache(bl_ctx *ctx, const bl_paged_cache &c, uint32_t dtype, uint32_t heads, uint32_t head_dim, bool written, const char *what) {
    if (!c.table || !c.lengths || !aligned(c.table, 4) || !aligned(c.lengths, 4))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: the cache's table or lengths are null or misaligned", what);
    if (c.pages == 0) return BL_OK;  // every page is missing
    const uint64_t width = row_bytes(c, dtype, head_dim), align = c.kind == BL_CACHE_INT4 ? 4 : 16;
    const bl_pages *const sides[] = {&c.k, &c.v};
    for (int n = 0; n < 2; n++) {
        const bl_pages &p = *sides[n];
        const char *name = n == 0 ? "keys" : "values";
        if (!p.data) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: the cache's %s are null", what, name);
        if (!aligned(p.data, align) || p.page_stride % align || p.row_stride % align || p.head_stride % align)
            return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the cache's %s: address or strides are not multiples of %llu bytes", what, name,
                          (unsigned long long)align);
        // Within a block of 16 rows, bytes are addressed by 32-bit offsets.
        if (p.row_stride > 1u << 24 || p.head_stride > 1ull << 40 || p.page_stride > 1ull << 40 ||
            (wide)p.page_stride * c.pages + (wide)p.row_stride * c.page_rows + (wide)p.head_stride * heads > (wide)1 << 62)
            return refuse(ctx, BL_ERR_TOO_LARGE, "%s: the strides of the cache's %s are too large", what, name);
        if (written && !steps_of(c, p, heads).apart(width)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: rows of %llu bytes of the cache's %s overlap", what,
                                                                          (unsigned long long)width, name);
    }
    if (!written) return BL_OK;
    // Keys and values side by side in one allocation: one more step of the same layout.
    if (overlap(extent_of(c, c.k, heads, width), extent_of(c, c.v, heads, width))) {
        const uint64_t k = (uint64_t)c.k.data, v = (uint64_t)c.v.data;
        Steps both = steps_of(c, c.k, heads);
        both.add(k < v ? v - k : k - v, 2);
        if (c.k.page_stride != c.v.page_stride || c.k.row_stride != c.v.row_stride || c.k.head_stride != c.v.head_stride || !both.apart(width))
            return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: the cache's keys and values overlap", what);
    }
    return BL_OK;
}

// Blocks beside the pages of both sides: the gaps between pages' rows are anyone's.
template <size_t N>
int check_blocks_beside_pages(bl_ctx *ctx, const bl_paged_cache &c, uint32_t heads, uint64_t width, const Named (&blocks)[N], const char *what) {
    if (c.pages == 0) return BL_OK;
    const bl_pages *const sides[] = {&c.k, &c.v};
    for (const Named &block : blocks)
        for (int n = 0; n < 2; n++) {
            if (block.bytes.rows == 0 || !overlap(block.bytes, extent_of(c, *sides[n], heads, width))) continue;
            Steps s = steps_of(c, *sides[n], heads);
            const wide from = (wide)block.bytes.at - (wide)(uint64_t)sides[n]->data;
            if (!s.apart(width) || meets(s, s.n, from, from + (wide)block.bytes.width, width))
                return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s overlaps the cache's %s", what, block.name, n == 0 ? "keys" : "values");
        }
    return BL_OK;
}
Named table_named(const bl_paged_cache &c, uint64_t documents) { return block_named(c.table, documents * c.max_pages * 4, "the cache's table"); }
Named lengths_named(const bl_paged_cache &c, uint64_t documents) { return block_named(c.lengths, documents * 4, "the cache's lengths"); }
Named offsets_named(const int32_t *offsets, uint64_t documents, const char *name) { return block_named(offsets, (documents + 1) * 4, name); }

int check_documents(bl_ctx *ctx, uint32_t documents, const int32_t *offsets, const char *what) {
    if (documents == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no documents", what);
    if (documents > 0x01000000u) return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u documents", what, documents);
    if (documents > 1 && !offsets) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u documents without offsets", what, documents);
    if (!aligned(offsets, 4)) return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the offsets are misaligned", what);
    return BL_OK;
}

// ---- attention ----

int check_paged(bl_ctx *ctx, const bl_paged_attention_args *a, const char *what) {
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->q_heads == 0 || a->kv_heads == 0 || a->q_heads % a->kv_heads)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u query heads over %u key heads", what, a->q_heads, a->kv_heads);
    if (int rc = check_cache_sizes(ctx, a->cache, a->head_dim, what)) return rc;
    if (a->documents == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no documents", what);
    if (a->mask != BL_MASK_NONE && a->mask != BL_MASK_CAUSAL) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: mask %u", what, a->mask);
    if (a->window && a->mask != BL_MASK_CAUSAL) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a window without a causal mask", what);
    if (!std::isfinite(a->scale)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: non-finite scale", what);
    if (!std::isfinite(a->softcap) || a->softcap < 0.0f)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a softcap that is negative or not finite", what);
    const float log2e = 1.4426950408889634f;
    if (!std::isfinite(a->scale * log2e) || !std::isfinite(a->softcap * log2e) || (a->softcap > 0.0f && !std::isfinite(2.0f * log2e * a->scale / a->softcap)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a scale of %g under a softcap of %g is beyond f32", what, a->scale, a->softcap);
    // 32-bit places of the (row, head of a group) pairs, and a grid of fewer than 2^32 threads
    // (a workgroup for each 16 of them and each key head at least; splits only where those are few).
    const uint64_t places = (uint64_t)a->q_rows * (a->q_heads / a->kv_heads);
    if (places > 0x40000000ull || a->documents > 0x01000000u || a->q_heads > 65535 || (places / 16 + a->documents) * a->kv_heads > 0xffffffull)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u query rows of %u heads, %u documents", what, a->q_rows, a->q_heads, a->documents);
    return BL_OK;
}

}  // namespace

extern "C" int bl_head_norm_rotary(bl_ctx *ctx, const bl_rotary_table *t, const bl_head_norm_args *a) {
    static const char *const what = "head norm";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_head_norm(ctx, a, what)) return rc;
    if (int rc = check_turn(ctx, t, a->positions, a->rows, a->head_dim, true, what)) return rc;
    const uint64_t size = element_size(a->dtype);
    if (int rc = check_weights(ctx, a->q_heads ? a->q_gamma : nullptr, size, what, "q_gamma")) return rc;
    if (int rc = check_weights(ctx, a->k_heads ? a->k_gamma : nullptr, size, what, "k_gamma")) return rc;
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, size};
    if (int rc = heads(a->q_in, a->rows, a->q_heads, false, "q_in")) return rc;
    if (int rc = heads(a->q_out, a->rows, a->q_heads, true, "q_out")) return rc;
    if (int rc = heads(a->k_in, a->rows, a->k_heads, false, "k_in")) return rc;
    if (int rc = heads(a->k_out, a->rows, a->k_heads, true, "k_out")) return rc;
    const auto named = [&](const bl_heads &h, uint32_t n, const char *name) { return heads_named(h, a->rows, n, a->head_dim, size, name); };
    const Named q_in = named(a->q_in, a->q_heads, "q_in"), q_out = named(a->q_out, a->q_heads, "q_out");
    const Named k_in = named(a->k_in, a->k_heads, "k_in"), k_out = named(a->k_out, a->k_heads, "k_out");
    if (int rc = check_apart(ctx, what, k_out, q_out)) return rc;
    if (int rc = check_in_place(ctx, what, q_out, a->q_out, q_in, a->q_in)) return rc;
    if (int rc = check_in_place(ctx, what, k_out, a->k_out, k_in, a->k_in)) return rc;
    if (int rc = check_apart(ctx, what, q_out, k_in)) return rc;
    if (int rc = check_apart(ctx, what, k_out, q_in)) return rc;
    for (const Named &out : {q_out, k_out})
        for (const Named &w : {weights_named(a->q_heads ? a->q_gamma : nullptr, a->head_dim, size, "q_gamma"), weights_named(a->k_heads ? a->k_gamma : nullptr, a->head_dim, size, "k_gamma")})
            if (w.bytes.at)
                if (int rc = check_apart(ctx, what, out, w)) return rc;
    if (int rc = check_outputs_apart(ctx, what, {q_out, k_out}, {positions_named(t, a->positions, a->rows)})) return rc;
    if (a->rows == 0) return BL_OK;
    bl::HeadsParams p = heads_params(t, a);
    Widest w(a->dtype);
    w.count(a->head_dim);
    w.count(p.table.pairs);
    w.heads(a->q_in, a->q_heads);
    w.heads(a->q_out, a->q_heads);
    w.heads(a->k_in, a->k_heads);
    w.heads(a->k_out, a->k_heads);
    w.vector(a->q_heads ? a->q_gamma : nullptr);
    w.vector(a->k_heads ? a->k_gamma : nullptr);
    p.vec = w.vec;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_heads_forward(p, a->dtype, bl_compute_units_of(ctx), bl_stream_of(ctx)), what);
}

extern "C" int bl_head_norm_rotary_backward_workspace(bl_ctx *ctx, const bl_head_norm_args *a, uint64_t *bytes) {
    static const char *const what = "head norm workspace";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!bytes) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no place for the answer", what);
    if (int rc = check_head_norm(ctx, a, what)) return rc;
    *bytes = heads_workspace(ctx, a);
    return BL_OK;
}

extern "C" int bl_head_norm_rotary_backward(bl_ctx *ctx, const bl_rotary_table *t, const bl_head_norm_args *a, const bl_head_norm_grads *g) {
    static const char *const what = "head norm backward";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_head_norm(ctx, a, what)) return rc;
    if (!g) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no gradients", what);
    if (int rc = check_turn(ctx, t, a->positions, a->rows, a->head_dim, true, what)) return rc;
    const uint64_t size = element_size(a->dtype);
    if (int rc = check_weights(ctx, a->q_heads ? a->q_gamma : nullptr, size, what, "q_gamma")) return rc;
    if (int rc = check_weights(ctx, a->k_heads ? a->k_gamma : nullptr, size, what, "k_gamma")) return rc;
    if (int rc = check_weights(ctx, g->d_q_gamma, 4, what, "d_q_gamma")) return rc;
    if (int rc = check_weights(ctx, g->d_k_gamma, 4, what, "d_k_gamma")) return rc;
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, size};
    if (int rc = heads(a->q_in, a->rows, a->q_heads, false, "q_in")) return rc;
    if (int rc = heads(g->dq_out, a->rows, a->q_heads, false, "dq_out")) return rc;
    if (int rc = heads(g->dq_in, a->rows, a->q_heads, true, "dq_in")) return rc;
    if (int rc = heads(a->k_in, a->rows, a->k_heads, false, "k_in")) return rc;
    if (int rc = heads(g->dk_out, a->rows, a->k_heads, false, "dk_out")) return rc;
    if (int rc = heads(g->dk_in, a->rows, a->k_heads, true, "dk_in")) return rc;
    const auto named = [&](const bl_heads &h, uint32_t n, const char *name) { return heads_named(h, a->rows, n, a->head_dim, size, name); };
    const Named q_in = named(a->q_in, a->q_heads, "q_in"), dq_out = named(g->dq_out, a->q_heads, "dq_out"), dq_in = named(g->dq_in, a->q_heads, "dq_in");
    const Named k_in = named(a->k_in, a->k_heads, "k_in"), dk_out = named(g->dk_out, a->k_heads, "dk_out"), dk_in = named(g->dk_in, a->k_heads, "dk_in");
    if (int rc = check_apart(ctx, what, dk_in, dq_in)) return rc;
    if (int rc = check_in_place(ctx, what, dq_in, g->dq_in, q_in, a->q_in)) return rc;
    if (int rc = check_in_place(ctx, what, dq_in, g->dq_in, dq_out, g->dq_out)) return rc;
    if (int rc = check_in_place(ctx, what, dk_in, g->dk_in, k_in, a->k_in)) return rc;
    if (int rc = check_in_place(ctx, what, dk_in, g->dk_in, dk_out, g->dk_out)) return rc;
    for (const Named &other : {k_in, dk_out})
        if (int rc = check_apart(ctx, what, dq_in, other)) return rc;
    for (const Named &other : {q_in, dq_out})
        if (int rc = check_apart(ctx, what, dk_in, other)) return rc;
    for (const Named &out : {dq_in, dk_in})
        for (const Named &w : {weights_named(a->q_heads ? a->q_gamma : nullptr, a->head_dim, size, "q_gamma"), weights_named(a->k_heads ? a->k_gamma : nullptr, a->head_dim, size, "k_gamma")})
            if (w.bytes.at)
                if (int rc = check_apart(ctx, what, out, w)) return rc;
    const uint64_t need = heads_workspace(ctx, a);
    if (g->workspace_bytes < need)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: a workspace of %llu bytes, %llu are needed", what, (unsigned long long)g->workspace_bytes,
                      (unsigned long long)need);
    if (!g->workspace || !aligned(g->workspace, 16))
        return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the workspace is null or not 16-byte aligned", what);
    if (int rc = check_outputs_apart(ctx, what, {dq_in, dk_in}, {positions_named(t, a->positions, a->rows)})) return rc;
    const Named floats[] = {block_named(a->q_heads ? g->d_q_gamma : nullptr, a->head_dim * 4, "d_q_gamma"),
                            block_named(a->k_heads ? g->d_k_gamma : nullptr, a->head_dim * 4, "d_k_gamma"), block_named(g->workspace, need, "the workspace")};
    if (int rc = check_outputs_apart(ctx, what, floats, {q_in, dq_out, dq_in, k_in, dk_out, dk_in})) return rc;
    bl::HeadsParams p = heads_params(t, a);
    p.dq_out = g->dq_out;
    p.dk_out = g->dk_out;
    p.dq_in = g->dq_in;
    p.dk_in = g->dk_in;
    p.d_q_gamma = a->q_heads ? g->d_q_gamma : nullptr;
    p.d_k_gamma = a->k_heads ? g->d_k_gamma : nullptr;
    p.partial = (float *)g->workspace;
    p.groups = heads_groups(ctx, a);
    Widest w(a->dtype);
    w.count(a->head_dim);
    w.count(p.table.pairs);
    w.heads(a->q_in, a->q_heads);
    w.heads(g->dq_out, a->q_heads);
    w.heads(g->dq_in, a->q_heads);
    w.heads(a->k_in, a->k_heads);
    w.heads(g->dk_out, a->k_heads);
    w.heads(g->dk_in, a->k_heads);
    w.vector(a->q_heads ? a->q_gamma : nullptr);
    w.vector(a->k_heads ? a->k_gamma : nullptr);
    p.vec = w.vec;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_heads_backward(p, a->dtype, bl_compute_units_of(ctx), bl_stream_of(ctx)), what);
}

extern "C" int bl_cache_append(bl_ctx *ctx, const bl_rotary_table *t, const bl_cache_append_args *a) {
    static const char *const what = "cache append";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->norm > BL_HEAD_NORM_CENTRED) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: norm %u", what, a->norm);
    if (a->norm != BL_HEAD_NORM_NONE && !finite_epsilon(a->epsilon))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: an epsilon that is negative or not finite", what);
    if (a->kv_heads == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no key heads", what);
    if (a->rows > 0x7fffffffu || a->q_heads > 65535 || a->kv_heads > 65535)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u rows of %u and %u heads", what, a->rows, a->q_heads, a->kv_heads);
    if (int rc = check_cache_sizes(ctx, a->cache, a->head_dim, what)) return rc;
    if (int rc = check_documents(ctx, a->documents, a->q_offsets, what)) return rc;
    if (int rc = check_turn(ctx, t, a->positions, a->rows, a->head_dim, t && t->axes > 1, what)) return rc;
    const uint64_t size = element_size(a->dtype);
    const void *const q_gamma = a->norm != BL_HEAD_NORM_NONE && a->q_heads ? a->q_gamma : nullptr;
    const void *const k_gamma = a->norm != BL_HEAD_NORM_NONE ? a->k_gamma : nullptr;
    if (int rc = check_weights(ctx, q_gamma, size, what, "q_gamma")) return rc;
    if (int rc = check_weights(ctx, k_gamma, size, what, "k_gamma")) return rc;
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, size};
    if (int rc = heads(a->q_in, a->rows, a->q_heads, false, "q_in")) return rc;
    if (int rc = heads(a->q_out, a->rows, a->q_heads, true, "q_out")) return rc;
    if (int rc = heads(a->k_in, a->rows, a->kv_heads, false, "k_in")) return rc;
    if (int rc = heads(a->v_in, a->rows, a->kv_heads, false, "v_in")) return rc;
    if (int rc = check_cache(ctx, a->cache, a->dtype, a->kv_heads, a->head_dim, true, what)) return rc;
    const auto named = [&](const bl_heads &h, uint32_t n, const char *name) { return heads_named(h, a->rows, n, a->head_dim, size, name); };
    const Named q_in = named(a->q_in, a->q_heads, "q_in"), q_out = named(a->q_out, a->q_heads, "q_out");
    const Named k_in = named(a->k_in, a->kv_heads, "k_in"), v_in = named(a->v_in, a->kv_heads, "v_in");
    if (int rc = check_in_place(ctx, what, q_out, a->q_out, q_in, a->q_in)) return rc;
    for (const Named &other : {k_in, v_in})
        if (int rc = check_apart(ctx, what, q_out, other)) return rc;
    const uint64_t width = row_bytes(a->cache, a->dtype, a->head_dim);
    for (const Named &side : {Named{extent_of(a->cache, a->cache.k, a->kv_heads, width), "the cache's keys"},
                              Named{extent_of(a->cache, a->cache.v, a->kv_heads, width), "the cache's values"}})
        for (const Named &other : {q_out, q_in, k_in, v_in})
            if (int rc = check_apart(ctx, what, side, other)) return rc;
    for (const Named &w : {weights_named(q_gamma, a->head_dim, size, "q_gamma"), weights_named(k_gamma, a->head_dim, size, "k_gamma")})
        if (w.bytes.at)
            if (int rc = check_apart(ctx, what, q_out, w)) return rc;
    const Named indices[] = {positions_named(t, a->positions, a->rows), offsets_named(a->q_offsets, a->documents, "q_offsets"),
                             table_named(a->cache, a->documents), lengths_named(a->cache, a->documents)};
    if (int rc = check_outputs_apart(ctx, what, {q_out}, indices)) return rc;
    if (int rc = check_blocks_beside_pages(ctx, a->cache, a->kv_heads, width, indices, what)) return rc;
    if (int rc = check_blocks_beside_pages(ctx, a->cache, a->kv_heads, width,
                                           {block_named(q_gamma, a->head_dim * size, "q_gamma"), block_named(k_gamma, a->head_dim * size, "k_gamma")}, what))
        return rc;
    if (a->rows == 0) return BL_OK;
    bl::AppendParams p{};
    if (t) p.h.table = *t;
    p.h.positions = a->positions;
    p.h.q_gamma = q_gamma;
    p.h.k_gamma = k_gamma;
    p.h.q_in = a->q_in;
    p.h.q_out = a->q_out;
    p.h.k_in = a->k_in;
    p.h.rows = a->rows;
    p.h.q_heads = a->q_heads;
    p.h.k_heads = a->kv_heads;
    p.h.head_dim = a->head_dim;
    p.h.norm = a->norm;
    p.h.epsilon = a->epsilon;
    p.v_in = a->v_in;
    p.cache = a->cache;
    p.q_offsets = a->q_offsets;
    p.documents = a->documents;
    Widest w(a->dtype);
    w.count(a->head_dim);
    w.count(p.h.table.pairs);
    w.heads(a->q_in, a->q_heads);
    w.heads(a->q_out, a->q_heads);
    w.heads(a->k_in, a->kv_heads);
    w.heads(a->v_in, a->kv_heads);
    w.vector(q_gamma);
    w.vector(k_gamma);
    p.h.vec = w.vec;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_cache_append(p, a->dtype, bl_compute_units_of(ctx), bl_stream_of(ctx)), what);
}

extern "C" int bl_cache_read(bl_ctx *ctx, const bl_cache_read_args *a) {
    static const char *const what = "cache read";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->kv_heads == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no key heads", what);
    if (a->rows > 0x7fffffffu || a->kv_heads > 65535) return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u rows of %u heads", what, a->rows, a->kv_heads);
    if (int rc = check_cache_sizes(ctx, a->cache, a->head_dim, what)) return rc;
    if (int rc = check_documents(ctx, a->documents, a->offsets, what)) return rc;
    if (!aligned(a->first, 4)) return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: first is misaligned", what);
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, 16};
    if (int rc = heads(a->k_out, a->rows, a->kv_heads, true, "k_out")) return rc;
    if (int rc = heads(a->v_out, a->rows, a->kv_heads, true, "v_out")) return rc;
    if (int rc = check_cache(ctx, a->cache, a->dtype, a->kv_heads, a->head_dim, false, what)) return rc;
    const uint64_t size = element_size(a->dtype), width = row_bytes(a->cache, a->dtype, a->head_dim);
    const Named k_out = heads_named(a->k_out, a->rows, a->kv_heads, a->head_dim, size, "k_out"), v_out = heads_named(a->v_out, a->rows, a->kv_heads, a->head_dim, size, "v_out");
    if (int rc = check_apart(ctx, what, v_out, k_out)) return rc;
    for (const Named &out : {k_out, v_out})
        for (const Named &side : {Named{extent_of(a->cache, a->cache.k, a->kv_heads, width), "the cache's keys"},
                                  Named{extent_of(a->cache, a->cache.v, a->kv_heads, width), "the cache's values"}})
            if (int rc = check_apart(ctx, what, out, side)) return rc;
    if (int rc = check_outputs_apart(ctx, what, {k_out, v_out}, {offsets_named(a->offsets, a->documents, "offsets"), block_named(a->first, a->documents * 4ull, "first"),
                                                                table_named(a->cache, a->documents), lengths_named(a->cache, a->documents)}))
        return rc;
    if (a->rows == 0) return BL_OK;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_cache_read(*a, bl_compute_units_of(ctx), bl_stream_of(ctx)), what);
}

extern "C" int bl_paged_attention_workspace(bl_ctx *ctx, const bl_paged_attention_args *a, uint64_t *bytes) {
    static const char *const what = "paged attention workspace";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!bytes) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no place for the answer", what);
    if (int rc = check_paged(ctx, a, what)) return rc;
    const bl::PagedPlan plan = bl::plan_paged(*a, bl_compute_units_of(ctx));
    *bytes = plan.partial_bytes + plan.stats_bytes;
    return BL_OK;
}

extern "C" int bl_paged_attention(bl_ctx *ctx, const bl_paged_attention_args *a) {
    static const char *const what = "paged attention";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_paged(ctx, a, what)) return rc;
    if (int rc = check_documents(ctx, a->documents, a->q_offsets, what)) return rc;
    if (!aligned(a->lse, 4)) return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: lse is misaligned", what);
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, 16};
    if (int rc = heads(a->q, a->q_rows, a->q_heads, false, "q")) return rc;
    if (int rc = heads(a->out, a->q_rows, a->q_heads, true, "out")) return rc;
    if (int rc = check_cache(ctx, a->cache, a->dtype, a->kv_heads, a->head_dim, false, what)) return rc;
    const uint64_t size = element_size(a->dtype), width = row_bytes(a->cache, a->dtype, a->head_dim);
    const Named out = heads_named(a->out, a->q_rows, a->q_heads, a->head_dim, size, "out");
    const Named q = heads_named(a->q, a->q_rows, a->q_heads, a->head_dim, size, "q");
    for (const Named &other : {q, Named{extent_of(a->cache, a->cache.k, a->kv_heads, width), "the cache's keys"},
                               Named{extent_of(a->cache, a->cache.v, a->kv_heads, width), "the cache's values"}})
        if (int rc = check_apart(ctx, what, out, other)) return rc;
    const bl::PagedPlan plan = bl::plan_paged(*a, bl_compute_units_of(ctx));
    const uint64_t need = plan.partial_bytes + plan.stats_bytes;
    if (a->workspace_bytes < need)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: a workspace of %llu bytes, %llu are needed", what, (unsigned long long)a->workspace_bytes,
                      (unsigned long long)need);
    if (need && (!a->workspace || !aligned(a->workspace, 16)))
        return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the workspace is null or not 16-byte aligned", what);
    if (int rc = check_outputs_apart(ctx, what, {out}, {offsets_named(a->q_offsets, a->documents, "q_offsets"), table_named(a->cache, a->documents),
                                                       lengths_named(a->cache, a->documents)}))
        return rc;
    const Named floats[] = {block_named(a->lse, (uint64_t)a->q_rows * a->q_heads * 4, "lse"), block_named(a->workspace, need, "the workspace")};
    if (int rc = check_outputs_apart(ctx, what, floats, {q, out})) return rc;
    if (int rc = check_blocks_beside_pages(ctx, a->cache, a->kv_heads, width, floats, what)) return rc;
    if (a->q_rows == 0) return BL_OK;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_paged(*a, plan, bl_stream_of(ctx)), what);
}
