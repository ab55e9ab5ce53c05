// The host side of the packed attention sublayer's operators
// (include/beatlm_ops.h): every check of a call's arguments, and the launch on
// the context's stream. Nothing here allocates or waits.
#include "ops.hpp"

#include "ops_checks.hpp"

using namespace bl::checks;

namespace {

// ---- LayerNorm ----

int check_norm(bl_ctx *ctx, const bl_layer_norm_args *a, const char *what) {
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->cols == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: zero columns", what);
    if (a->cols > BL_LAYER_NORM_MAX_COLS)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u columns, at most %u", what, a->cols, BL_LAYER_NORM_MAX_COLS);
    if (a->rows > 0x7fffffffu) return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u rows", what, a->rows);
    return BL_OK;
}

// A row-strided tensor of the call: there, its rows apart, its elements aligned.
int check_rows(bl_ctx *ctx, const bl_layer_norm_args *a, const void *p, uint64_t stride, const char *what, const char *name) {
    if (a->rows == 0) return BL_OK;
    if (!p) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
    if (stride < a->cols)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s's rows of %u are %llu elements apart", what, name, a->cols, (unsigned long long)stride);
    if (!aligned(p, element_size(a->dtype))) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is misaligned", what, name);
    return BL_OK;
}

Named rows_named(const bl_layer_norm_args *a, const void *p, uint64_t stride, const char *name) {
    return {bytes_of({(void *)p, stride, 0}, a->rows, 1, a->cols, element_size(a->dtype)), name};
}
Named vector_named(const bl_layer_norm_args *a, const void *p, const char *name) { return {bytes_of({(void *)p, 0, 0}, 1, 1, a->cols, element_size(a->dtype)), name}; }

uint64_t norm_workspace(bl_ctx *ctx, const bl_layer_norm_args *a) {
    return (uint64_t)bl::norm_groups(a->rows, a->cols, bl_compute_units_of(ctx), bl::NORM_BACKWARD_GROUPS) * 2 * a->cols * sizeof(float);
}

// ---- attention ----

int check_attention(bl_ctx *ctx, const bl_packed_attention_args *a, const char *what) {
    if (!a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (a->q_heads == 0 || a->kv_heads == 0 || a->q_heads % a->kv_heads)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u query heads over %u key heads", what, a->q_heads, a->kv_heads);
    if (a->head_dim == 0 || a->head_dim % 8 || a->head_dim > BL_ATTENTION_MAX_HEAD_DIM)
        return refuse(ctx, a->head_dim > BL_ATTENTION_MAX_HEAD_DIM ? BL_ERR_TOO_LARGE : BL_ERR_INVALID_ARGUMENT,
                      "%s: heads of %u, not a multiple of 8 up to %u", what, a->head_dim, BL_ATTENTION_MAX_HEAD_DIM);
    if (a->documents == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no documents", what);
    if (a->mask > BL_MASK_PREFIX) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown mask %u", what, a->mask);
    if (a->axes > 3) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u axes, at most 3", what, a->axes);
    if (!std::isfinite(a->scale)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: non-finite scale", what);
    if (!std::isfinite(a->softcap) || a->softcap < 0.0f)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a softcap that is negative or not finite", what);
    // What the scores are multiplied by, in base two and under the cap.
    const float log2e = 1.4426950408889634f;
    if (!std::isfinite(a->scale * log2e) || !std::isfinite(a->softcap * log2e) || (a->softcap > 0.0f && !std::isfinite(2.0f * log2e * a->scale / a->softcap)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a scale of %g under a softcap of %g is beyond f32", what, a->scale, a->softcap);
    // 32-bit places of the (row, head of a group) pairs, and of the tiles with one more per document.
    // A grid has a workgroup of up to 512 threads for each 128 of them and each
    // key head (splits only where those are few), and fewer than 2^32 threads.
    const uint64_t places = (uint64_t)a->q_rows * (a->q_heads / a->kv_heads);
    const uint64_t most = (places > a->k_rows ? places : a->k_rows) / 128 + a->documents;
    if (places > 0x40000000ull || a->k_rows > 0x40000000u || a->documents > 0x01000000u || a->q_heads > 65535 || most * a->kv_heads > 0x7fffffull)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u query rows of %u heads, %u key rows, %u documents", what, a->q_rows, a->q_heads,
                      a->k_rows, a->documents);
    return BL_OK;
}

Named q_named(const bl_packed_attention_args *a, const bl_heads &h, const char *name) {
    return {bytes_of(h, a->q_rows, a->q_heads, a->head_dim, element_size(a->dtype)), name};
}
Named k_named(const bl_packed_attention_args *a, const bl_heads &h, const char *name) {
    return {bytes_of(h, a->k_rows, a->kv_heads, a->head_dim, element_size(a->dtype)), name};
}

// What the kernels will read, beyond the sizes.
int check_attention_arrays(bl_ctx *ctx, const bl_packed_attention_args *a, const char *what) {
    const bool packed = a->q_offsets != nullptr;
    if (!a->k_begin != !a->k_end) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: k_begin without k_end, or the other way round", what);
    if (a->documents > 1 && (!packed || !a->k_begin))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u documents without offsets", what, a->documents);
    if (a->mask == BL_MASK_PREFIX && !a->prefix) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a prefix mask without prefixes", what);
    if (a->axes && !a->slopes) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: positions without slopes", what);
    if (a->axes && ((a->q_rows && !a->q_positions) || (a->k_rows && !a->k_positions)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %u axes without positions", what, a->axes);
    const void *words[] = {a->q_offsets, a->k_begin, a->k_end, a->prefix, a->slopes, a->q_positions, a->k_positions, a->lse};
    for (const void *w : words)
        if (!aligned(w, 4)) return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: a 32-bit array is misaligned", what);
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, 16};
    if (int rc = heads(a->q, a->q_rows, a->q_heads, false, "q")) return rc;
    if (int rc = heads(a->k, a->k_rows, a->kv_heads, false, "k")) return rc;
    if (int rc = heads(a->v, a->k_rows, a->kv_heads, false, "v")) return rc;
    return heads(a->out, a->q_rows, a->q_heads, true, "out");
}

int check_workspace(bl_ctx *ctx, const bl_packed_attention_args *a, uint64_t need, const char *what) {
    if (a->workspace_bytes < need)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: a workspace of %llu bytes, %llu are needed", what, (unsigned long long)a->workspace_bytes,
                      (unsigned long long)need);
    if (need && (!a->workspace || !aligned(a->workspace, 16)))
        return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the workspace is null or not 16-byte aligned", what);
    return BL_OK;
}

}  // namespace

extern "C" int bl_layer_norm(bl_ctx *ctx, const bl_layer_norm_args *a) {
    static const char *const what = "layer norm";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_norm(ctx, a, what)) return rc;
    if (!std::isfinite(a->epsilon) || a->epsilon < 0.0f)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: an epsilon that is negative or not finite", what);
    const uint64_t size = element_size(a->dtype);
    if (int rc = check_rows(ctx, a, a->x, a->x_stride, what, "x")) return rc;
    if (int rc = check_rows(ctx, a, a->y, a->y_stride, what, "y")) return rc;
    if (int rc = check_vector(ctx, a->gamma, size, what, "gamma")) return rc;
    if (int rc = check_vector(ctx, a->beta, size, what, "beta")) return rc;
    if (!aligned(a->mean, 4) || !aligned(a->rstd, 4)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: the statistics are misaligned", what);
    if (a->x == a->y && a->x_stride != a->y_stride && a->rows > 1)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: y is x with another stride", what);
    const Named y = rows_named(a, a->y, a->y_stride, "y");
    if (a->x != a->y)
        if (int rc = check_apart(ctx, what, y, rows_named(a, a->x, a->x_stride, "x"))) return rc;
    if (int rc = check_apart(ctx, what, y, vector_named(a, a->gamma, "gamma"))) return rc;
    if (int rc = check_apart(ctx, what, y, vector_named(a, a->beta, "beta"))) return rc;
    if (a->rows == 0) return BL_OK;
    bl::NormParams p{};
    p.x = a->x;
    p.gamma = a->gamma;
    p.beta = a->beta;
    p.y = a->y;
    p.mean = a->mean;
    p.rstd = a->rstd;
    p.x_stride = a->x_stride;
    p.y_stride = a->y_stride;
    p.rows = a->rows;
    p.cols = a->cols;
    p.epsilon = a->epsilon;
    p.groups = bl::norm_groups(a->rows, a->cols, bl_compute_units_of(ctx), bl::NORM_FORWARD_GROUPS);
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_norm_forward(p, a->dtype, bl_stream_of(ctx)), what);
}

extern "C" int bl_layer_norm_backward_workspace(bl_ctx *ctx, const bl_layer_norm_args *a, uint64_t *bytes) {
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!bytes) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "layer norm workspace: no place for the answer");
    if (int rc = check_norm(ctx, a, "layer norm workspace")) return rc;
    *bytes = norm_workspace(ctx, a);
    return BL_OK;
}

extern "C" int bl_layer_norm_backward(bl_ctx *ctx, const bl_layer_norm_args *a, const bl_layer_norm_grads *g) {
    static const char *const what = "layer norm backward";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_norm(ctx, a, what)) return rc;
    if (!g) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no gradients", what);
    const uint64_t size = element_size(a->dtype);
    if (int rc = check_rows(ctx, a, a->x, a->x_stride, what, "x")) return rc;
    if (int rc = check_rows(ctx, a, g->dy, g->dy_stride, what, "dy")) return rc;
    if (int rc = check_rows(ctx, a, g->dx, g->dx_stride, what, "dx")) return rc;
    if (int rc = check_vector(ctx, a->gamma, size, what, "gamma")) return rc;
    if (int rc = check_vector(ctx, g->d_gamma, 4, what, "d_gamma")) return rc;
    if (int rc = check_vector(ctx, g->d_beta, 4, what, "d_beta")) return rc;
    if (a->rows) {
        if (int rc = check_vector(ctx, a->mean, 4, what, "mean")) return rc;
        if (int rc = check_vector(ctx, a->rstd, 4, what, "rstd")) return rc;
    }
    if (a->rows > 1 && ((g->dx == a->x && g->dx_stride != a->x_stride) || (g->dx == g->dy && g->dx_stride != g->dy_stride)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: dx is x or dy with another stride", what);
    const Named dx = rows_named(a, g->dx, g->dx_stride, "dx");
    if (g->dx != a->x)
        if (int rc = check_apart(ctx, what, dx, rows_named(a, a->x, a->x_stride, "x"))) return rc;
    if (g->dx != g->dy)
        if (int rc = check_apart(ctx, what, dx, rows_named(a, g->dy, g->dy_stride, "dy"))) return rc;
    if (int rc = check_apart(ctx, what, dx, vector_named(a, a->gamma, "gamma"))) return rc;
    const uint64_t need = norm_workspace(ctx, a);
    if (g->workspace_bytes < need)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: a workspace of %llu bytes, %llu are needed", what, (unsigned long long)g->workspace_bytes,
                      (unsigned long long)need);
    if (need && (!g->workspace || !aligned(g->workspace, 16)))
        return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: the workspace is null or not 16-byte aligned", what);
    bl::NormParams p{};
    p.x = a->x;
    p.gamma = a->gamma;
    p.dy = g->dy;
    p.dx = g->dx;
    p.mean = a->mean;
    p.rstd = a->rstd;
    p.d_gamma = g->d_gamma;
    p.d_beta = g->d_beta;
    p.partial = (float *)g->workspace;
    p.x_stride = a->x_stride;
    p.dy_stride = g->dy_stride;
    p.dx_stride = g->dx_stride;
    p.rows = a->rows;
    p.cols = a->cols;
    p.groups = bl::norm_groups(a->rows, a->cols, bl_compute_units_of(ctx), bl::NORM_BACKWARD_GROUPS);
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_norm_backward(p, a->dtype, bl_stream_of(ctx)), what);
}

extern "C" int bl_rotary_table_make(const uint32_t *sections, uint32_t axes, double base, uint32_t ladder, uint32_t layout,
                                    bl_rotary_table *out) {
    if (!sections || !out || axes == 0 || axes > 3 || ladder > BL_ROTARY_PER_AXIS || layout > BL_ROTARY_NEIGHBOURS)
        return BL_ERR_INVALID_ARGUMENT;
    if (!std::isfinite(base) || base <= 0.0) return BL_ERR_INVALID_ARGUMENT;
    uint64_t pairs = 0;
    for (uint32_t a = 0; a < axes; a++) pairs += sections[a];
    if (pairs == 0 || pairs > BL_ROTARY_MAX_PAIRS) return BL_ERR_INVALID_ARGUMENT;
    *out = bl_rotary_table{};
    out->axes = axes;
    out->pairs = (uint32_t)pairs;
    out->layout = layout;
    uint32_t at = 0;
    for (uint32_t a = 0; a < axes; a++)
        for (uint32_t i = 0; i < sections[a]; i++, at++) {
            const double share = ladder == BL_ROTARY_SHARED ? (double)at / (double)pairs : (double)i / (double)sections[a];
            out->turns[at] = std::pow(base, -share) / (2.0 * M_PI);
            out->axis[at] = (uint8_t)a;
        }
    return BL_OK;
}

extern "C" int bl_rotary(bl_ctx *ctx, const bl_rotary_table *t, const bl_rotary_args *a) {
    static const char *const what = "rotary positions";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!t || !a) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no table or no arguments", what);
    if (!known(a->dtype)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %u", what, a->dtype);
    if (int rc = check_table(ctx, t, a->head_dim, what)) return rc;
    if (a->inverse > 1) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: inverse is 0 or 1", what);
    if (a->q_heads == 0 && a->k_heads == 0) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no heads", what);
    if (a->rows > 0x7fffffffu || a->q_heads > 65535 || a->k_heads > 65535)
        return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %u rows of %u and %u heads", what, a->rows, a->q_heads, a->k_heads);
    if (a->rows && (!a->positions || !aligned(a->positions, 4)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: positions are null or misaligned", what);
    const uint64_t size = element_size(a->dtype);
    if ((a->q_heads && a->q_in.data && a->q_in.data == a->q_out.data && !same_heads(a->q_in, a->q_out)) ||
        (a->k_heads && a->k_in.data && a->k_in.data == a->k_out.data && !same_heads(a->k_in, a->k_out)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: an output is its input with other strides", what);
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, size};
    if (int rc = heads(a->q_in, a->rows, a->q_heads, false, "q_in")) return rc;
    if (int rc = heads(a->q_out, a->rows, a->q_heads, true, "q_out")) return rc;
    if (int rc = heads(a->k_in, a->rows, a->k_heads, false, "k_in")) return rc;
    if (int rc = heads(a->k_out, a->rows, a->k_heads, true, "k_out")) return rc;
    const auto named = [&](const bl_heads &h, uint32_t n, const char *name) { return Named{bytes_of(h, a->rows, n, a->head_dim, size), name}; };
    const Named q_in = named(a->q_in, a->q_heads, "q_in"), q_out = named(a->q_out, a->q_heads, "q_out");
    const Named k_in = named(a->k_in, a->k_heads, "k_in"), k_out = named(a->k_out, a->k_heads, "k_out");
    if (int rc = check_apart(ctx, what, k_out, q_out)) return rc;
    if (!same_heads(a->q_in, a->q_out))
        if (int rc = check_apart(ctx, what, q_out, q_in)) return rc;
    if (!same_heads(a->k_in, a->k_out))
        if (int rc = check_apart(ctx, what, k_out, k_in)) return rc;
    if (a->q_in.data != a->k_in.data) {  // one input given as both is the host's to order
        if (int rc = check_apart(ctx, what, q_out, k_in)) return rc;
        if (int rc = check_apart(ctx, what, k_out, q_in)) return rc;
    }
    if (a->rows == 0) return BL_OK;
    bl::RotaryParams p{};
    p.table = *t;
    p.positions = a->positions;
    p.q_in = a->q_in;
    p.q_out = a->q_out;
    p.k_in = a->k_in;
    p.k_out = a->k_out;
    p.rows = a->rows;
    p.q_heads = a->q_heads;
    p.k_heads = a->k_heads;
    p.head_dim = a->head_dim;
    p.sign = a->inverse ? -1.0f : 1.0f;
    p.copy_q = !same_heads(a->q_in, a->q_out);
    p.copy_k = !same_heads(a->k_in, a->k_out);
    // 16-byte chunks: the pairs, the copied tail and every head start at them.
    const uint64_t lanes = 16 / size;
    const auto chunked = [&](const bl_heads &h, uint32_t n) {
        return n == 0 || (aligned(h.data, 16) && h.row_stride % lanes == 0 && h.head_stride % lanes == 0);
    };
    p.vector = t->pairs % lanes == 0 && a->head_dim % lanes == 0 && chunked(a->q_in, a->q_heads) && chunked(a->q_out, a->q_heads) &&
               chunked(a->k_in, a->k_heads) && chunked(a->k_out, a->k_heads);
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_rotary(p, a->dtype, bl_compute_units_of(ctx), bl_stream_of(ctx)), what);
}

extern "C" int bl_packed_attention_workspace(bl_ctx *ctx, const bl_packed_attention_args *a, uint32_t backward, uint64_t *bytes) {
    static const char *const what = "packed attention workspace";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (!bytes || backward > 1) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no place for the answer, or backward not 0 or 1", what);
    if (int rc = check_attention(ctx, a, what)) return rc;
    const bl::PackedPlan plan = bl::plan_packed(*a, bl_compute_units_of(ctx));
    *bytes = backward && plan.backward_bytes > plan.forward_bytes ? plan.backward_bytes : plan.forward_bytes;
    return BL_OK;
}

extern "C" int bl_packed_attention(bl_ctx *ctx, const bl_packed_attention_args *a) {
    static const char *const what = "packed attention";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_attention(ctx, a, what)) return rc;
    if (int rc = check_attention_arrays(ctx, a, what)) return rc;
    const Named out[] = {q_named(a, a->out, "out")}, in[] = {q_named(a, a->q, "q"), k_named(a, a->k, "k"), k_named(a, a->v, "v")};
    if (int rc = check_separate(ctx, what, out, in)) return rc;
    const bl::PackedPlan plan = bl::plan_packed(*a, bl_compute_units_of(ctx));
    if (int rc = check_workspace(ctx, a, plan.forward_bytes, what)) return rc;
    if (a->q_rows == 0) return BL_OK;
    bl::PackedParams p{};
    p.a = *a;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_packed_forward(p, plan, bl_stream_of(ctx)), what);
}

extern "C" int bl_packed_attention_backward(bl_ctx *ctx, const bl_packed_attention_args *a, const bl_packed_attention_grads *g) {
    static const char *const what = "packed attention backward";
    if (!ctx) return BL_ERR_INVALID_ARGUMENT;
    if (int rc = check_attention(ctx, a, what)) return rc;
    if (!g) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: no gradients", what);
    if (int rc = check_attention_arrays(ctx, a, what)) return rc;
    if (a->k_begin && a->k_end != a->k_begin + 1)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: the keys are not packed by one array of offsets (k_end = k_begin + 1)", what);
    if (a->q_rows && !a->lse) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: lse is null", what);
    if (g->d_slopes && (!a->slopes || !aligned(g->d_slopes, 4)))
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: d_slopes without slopes, or misaligned", what);
    const HeadsCheck heads{ctx, what, a->dtype, a->head_dim, 16};
    if (int rc = heads(g->d_out, a->q_rows, a->q_heads, false, "d_out")) return rc;
    if (int rc = heads(g->d_q, a->q_rows, a->q_heads, true, "d_q")) return rc;
    if (int rc = heads(g->d_k, a->k_rows, a->kv_heads, true, "d_k")) return rc;
    if (int rc = heads(g->d_v, a->k_rows, a->kv_heads, true, "d_v")) return rc;
    const Named grads[] = {q_named(a, g->d_q, "d_q"), k_named(a, g->d_k, "d_k"), k_named(a, g->d_v, "d_v")};
    const Named in[] = {q_named(a, a->q, "q"), k_named(a, a->k, "k"), k_named(a, a->v, "v"), q_named(a, a->out, "out"), q_named(a, g->d_out, "d_out")};
    if (int rc = check_separate(ctx, what, grads, in)) return rc;
    const bl::PackedPlan plan = bl::plan_packed(*a, bl_compute_units_of(ctx));
    if (int rc = check_workspace(ctx, a, plan.backward_bytes, what)) return rc;
    bl::PackedParams p{};
    p.a = *a;
    p.g = *g;
    const DeviceScope scope(bl_device_of(ctx));
    if (scope.status != hipSuccess) return launched(ctx, scope.status, what);
    return launched(ctx, bl::launch_packed_backward(p, plan, bl_stream_of(ctx)), what);
}
