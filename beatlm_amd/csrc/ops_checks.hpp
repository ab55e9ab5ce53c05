// What the packed sublayer's operators check alike on the host
// (include/beatlm_ops.h): refusals, strided tensors, and that what a call writes
// lies apart from what it reads.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/beatlm_ops.h"
#include "ctx.hpp"

namespace bl {
namespace checks {

inline int refuse(bl_ctx *ctx, int code, const char *fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return bl_fail(ctx, code, msg);
}

inline uint64_t element_size(uint32_t dtype) { return dtype == BL_F32 ? 4 : 2; }
inline bool known(uint32_t dtype) { return dtype == BL_F32 || dtype == BL_F16 || dtype == BL_BF16; }
inline bool aligned(const void *p, uint64_t bytes) { return (uintptr_t)p % bytes == 0; }

inline int launched(bl_ctx *ctx, hipError_t e, const char *what) {
    return e == hipSuccess ? BL_OK : refuse(ctx, BL_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// ---- what a call writes lies apart ----

// The bytes of a strided tensor: `rows` by `heads` pieces of `width`, steps in bytes.
struct Bytes {
    uint64_t at, row, rows, head, heads, width;
};
typedef __int128 wide;  // products of a call's strides and counts

inline Bytes bytes_of(const bl_heads &h, uint64_t rows, uint64_t heads, uint64_t head_dim, uint64_t size) {
    return {(uint64_t)h.data, h.row_stride * size, rows, h.head_stride * size, heads, head_dim * size};
}

// The least n >= 0 with n * step mod m in [lo, hi] (0 < lo <= hi < m), or -1.
inline wide first_within(wide step, wide m, wide lo, wide hi) {
    if (step == 0) return -1;
    if (2 * step > m) return first_within(m - step, m, m - hi, m - lo);  // counted downwards
    const wide n = (lo + step - 1) / step;
    if (n * step <= hi) return n;
    // No multiple of step in [lo, hi]: so many times round m that one comes to lie in it.
    const wide round = first_within((step - m % step) % step, step, lo % step, hi % step);
    return round < 0 ? -1 : (lo + m * round + step - 1) / step;
}

// Whether two rows of pieces meet: from + x p of width w and y q of width v,
// x < n, y < k.
inline bool rows_meet(wide from, wide p, wide n, wide w, wide q, wide k, wide v) {
    if (p == 0) n = 1;
    if (q == 0) k = 1;
    if (k == 1) q = n * p + w + v + (from < 0 ? -from : from);  // any step beyond the rest
    // A y serves where y q lies in [t - room, t], t = from + x p + w - 1.
    const wide t0 = from + w - 1, room = w + v - 2;
    const wide most = (k - 1) * q + room - t0;  // x p is no more than this, and t no less than 0
    if (most < 0 || (p == 0 && t0 < 0)) return false;
    const wide first = t0 >= 0 ? 0 : (-t0 + p - 1) / p, last = p == 0 ? 0 : most / p < n - 1 ? most / p : n - 1;
    if (first > last) return false;
    if (room >= q - 1) return true;
    const wide at = (t0 + first * p) % q;
    if (at <= room) return true;
    const wide steps = first_within(p % q, q, q - at, q - at + room);
    return steps >= 0 && steps <= last - first;
}

inline bool overlap(Bytes a, Bytes b) {
    for (Bytes *t : {&a, &b}) {
        if (t->rows == 0 || t->heads == 0) return false;
        if (t->head == 0) t->heads = 1;
        if (t->row == 0) t->rows = 1;
        // Pieces that lie end to end are one.
        if (t->heads > 1 && t->head == t->width) t->width *= t->heads, t->heads = 1;
        if (t->rows > 1 && t->row == t->width) t->width *= t->rows, t->rows = 1;
        if (t->heads > 1 && t->head == t->width) t->width *= t->heads, t->heads = 1;
    }
    const auto end = [](const Bytes &t) { return (wide)t.at + (wide)t.row * (t.rows - 1) + (wide)t.head * (t.heads - 1) + t.width; };
    if (end(a) <= (wide)b.at || end(b) <= (wide)a.at) return false;
    // As a rule all heads of a row lie beside all of the other's: one look at
    // them as one piece.
    const auto all = [](const Bytes &t) { return (wide)t.head * (t.heads - 1) + t.width; };
    if (!rows_meet((wide)a.at - (wide)b.at, a.row, a.rows, all(a), b.row, b.rows, all(b))) return false;
    const auto meet = [&](wide heads_apart) {
        return rows_meet((wide)a.at - (wide)b.at + heads_apart, a.row, a.rows, a.width, b.row, b.rows, b.width);
    };
    if (a.heads == 1 || b.heads == 1 || a.head == b.head) {  // heads by their difference alone
        const wide step = a.heads == 1 ? b.head : a.head;
        for (wide d = 1 - (wide)b.heads; d < (wide)a.heads; d++)
            if (meet(d * step)) return true;
        return false;
    }
    if (a.heads * b.heads > 1u << 20) return true;  // too many pairs to look at, of rows that do meet
    for (wide x = 0; x < (wide)a.heads; x++)
        for (wide y = 0; y < (wide)b.heads; y++)
            if (meet(x * a.head - y * (wide)b.head)) return true;
    return false;
}

struct Named {
    Bytes bytes;
    const char *name;
};
inline int check_apart(bl_ctx *ctx, const char *what, const Named &written, const Named &other) {
    if (!overlap(written.bytes, other.bytes)) return BL_OK;
    const bool same = written.bytes.at == other.bytes.at;
    return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s %s %s", what, written.name, same ? "is" : "overlaps", other.name);
}

inline int check_vector(bl_ctx *ctx, const void *p, uint64_t size, const char *what, const char *name) {
    if (!p) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
    if (!aligned(p, size)) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is misaligned", what, name);
    return BL_OK;
}

// ---- views [rows][heads][head_dim] ----

struct HeadsCheck {
    bl_ctx *ctx;
    const char *what;
    uint32_t dtype, head_dim;
    uint64_t align;  // bytes the address and both strides are multiples of

    int operator()(const bl_heads &h, uint32_t rows, uint32_t heads, bool written, const char *name) const {
        if (rows == 0 || heads == 0) return BL_OK;
        if (!h.data) return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
        const uint64_t size = element_size(dtype);
        if (!aligned(h.data, align) || (rows > 1 && h.row_stride * size % align) || (heads > 1 && h.head_stride * size % align))
            return refuse(ctx, BL_ERR_MISALIGNED_PLACEMENT, "%s: %s's address or strides are not multiples of %llu bytes", what, name,
                          (unsigned long long)align);
        // Rows of all heads, or heads of all rows: either lies in one step of the other.
        const auto apart = [&](uint64_t step, uint64_t n, uint64_t inner, uint64_t m) {
            return n <= 1 || (step >= head_dim && (m <= 1 || inner > step || step >= (m - 1) * inner + head_dim));
        };
        if (written && (!apart(h.row_stride, rows, h.head_stride, heads) || !apart(h.head_stride, heads, h.row_stride, rows)))
            return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: %s's heads of %u overlap", what, name, head_dim);
        // Within a tile of 128 rows, bytes are addressed by 32-bit offsets.
        if ((rows > 1 && h.row_stride > (1u << 24) / size) || (heads > 1 && h.head_stride > (1ull << 40)))
            return refuse(ctx, BL_ERR_TOO_LARGE, "%s: %s's strides are too large", what, name);
        return BL_OK;
    }
};

// Tensors that a call writes share nothing with each other or with those it reads.
template <size_t N, size_t M>
inline int check_separate(bl_ctx *ctx, const char *what, const Named (&written)[N], const Named (&read)[M]) {
    for (size_t i = 0; i < N; i++)
        for (size_t j = 0; j < i + M; j++)
            if (int rc = check_apart(ctx, what, written[i], j < i ? written[j] : read[j - i])) return rc;
    return BL_OK;
}

// A table that the kernels can follow, for heads of head_dim.
inline int check_table(bl_ctx *ctx, const bl_rotary_table *t, uint32_t head_dim, const char *what) {
    if (t->axes == 0 || t->axes > 3 || t->pairs == 0 || t->pairs > BL_ROTARY_MAX_PAIRS || t->layout > BL_ROTARY_NEIGHBOURS)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: a table of %u axes, %u pairs, layout %u", what, t->axes, t->pairs, t->layout);
    for (uint32_t i = 0; i < t->pairs; i++)
        if (t->axis[i] >= t->axes || !std::isfinite(t->turns[i]))
            return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: pair %u turns by axis %u of %u, or by no finite frequency", what, i, t->axis[i], t->axes);
    if (head_dim < 2 * t->pairs || head_dim > 2 * BL_ROTARY_MAX_PAIRS)
        return refuse(ctx, BL_ERR_INVALID_ARGUMENT, "%s: heads of %u for %u pairs", what, head_dim, t->pairs);
    return BL_OK;
}

inline bool same_heads(const bl_heads &x, const bl_heads &y) {
    return x.data == y.data && x.row_stride == y.row_stride && x.head_stride == y.head_stride;
}

}  // namespace checks
}  // namespace bl
