/*
 * beatlm HIP backend: norms of each head of queries and keys with their rotary
 * positions, and a cache of keys and values in pages, of the tensors' type or
 * of 4-bit codes, with what appends to it, reads it back and attends over it,
 * as direct calls over device pointers. They stand beside beatlm_ops.h's rotary
 * positions and packed attention, for hosts whose models norm their heads and
 * that decode many sequences whose lengths they do not know beforehand. The
 * reference has no counterpart: it runs one image at a time, without a cache.
 *
 * Conventions are beatlm_ops.h's: statuses, the context's stream and device,
 * nothing allocated and nothing waited for, argument structs read during the
 * call alone and device arrays when the kernels run, a workspace for each call
 * that may overlap another, and a refused call launches nothing.
 *
 * Tensors and pages that a call writes share no byte with what else it reads or
 * writes, other than where an output may be an input itself, and lse, weights'
 * gradients and a workspace none with tensors and pages: such a call is refused.
 * Not looked at, and the host's to keep apart: lse, gradients and workspace
 * beside each other and beside weights and index arrays, and what the device
 * arrays say (two rows of a call for one row of a page).
 */
#ifndef BEATLM_CACHE_H
#define BEATLM_CACHE_H

#include "beatlm_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------
 * Norms of each head of queries and keys, with their rotary positions
 *
 * For each row and head, over the head's channels c:
 *   RMS:      n = x rstd,               rstd = 1 / sqrt(mean_c(x^2) + epsilon)
 *   CENTRED:  n = (x - mean_c(x)) rstd, rstd = 1 / sqrt(mean_c((x - mean)^2) + epsilon)
 *   z = n gamma,  y = z turned as bl_rotary turns it
 * rounded once, at the end. gamma is the queries' or the keys' and shared by
 * their heads.
 *
 *   dz = dy turned back,  d_gamma = sum over rows and heads of dz n,  g = dz gamma
 *   dx = rstd (g - n mean_c(g n)), and CENTRED: less rstd mean_c(g)
 *
 * Sums and statistics are f32; the sums over rows are made in a fixed order, so
 * equal calls give equal bits. The backward makes the statistics again from x.
 * rows = 0 writes nothing but zeros to the weights' gradients.
 * ------------------------------------------------------------------------ */
#define BL_HEAD_NORM_MAX_HEAD_DIM 256u
enum { BL_HEAD_NORM_NONE = 0, BL_HEAD_NORM_RMS = 1, BL_HEAD_NORM_CENTRED = 2 };

typedef struct {
    uint32_t dtype;
    uint32_t rows;
    uint32_t q_heads, k_heads;  /* either may be 0: that tensor and its weights are not touched */
    uint32_t head_dim;          /* 2 * the table's pairs to BL_HEAD_NORM_MAX_HEAD_DIM */
    uint32_t norm;              /* BL_HEAD_NORM_RMS or _CENTRED (NONE is bl_rotary) */
    float epsilon;              /* >= 0, finite */
    const int32_t *positions;   /* [rows][axes]; not read without a table */
    const void *q_gamma, *k_gamma; /* [head_dim] of `dtype`, or NULL: ones */
    bl_heads q_in, q_out, k_in, k_out; /* out may be in itself (the same strides); the backward does not use out */
} bl_head_norm_args;

typedef struct {
    bl_heads dq_out, dk_out;    /* gradients of q_out and k_out, read */
    bl_heads dq_in, dk_in;      /* of q_in and k_in, written; may be dq_out or q_in itself (the same strides) */
    float *d_q_gamma, *d_k_gamma; /* [head_dim], or NULL: not wanted */
    void *workspace;            /* 16-byte aligned */
    uint64_t workspace_bytes;
} bl_head_norm_grads;

/* table NULL: norms alone. */
int bl_head_norm_rotary(bl_ctx *ctx, const bl_rotary_table *table, const bl_head_norm_args *args);
int bl_head_norm_rotary_backward_workspace(bl_ctx *ctx, const bl_head_norm_args *args, uint64_t *bytes);
int bl_head_norm_rotary_backward(bl_ctx *ctx, const bl_rotary_table *table, const bl_head_norm_args *args, const bl_head_norm_grads *grads);

/* ------------------------------------------------------------------------
 * A cache of keys and values in pages
 *
 * A page holds page_rows tokens of every key head; document d's key j is row
 * j % page_rows of the page table[d][j / page_rows]. The row of (page, row,
 * head) starts at data + page * page_stride + row * row_stride + head *
 * head_stride bytes, so pages may be laid out head by head or token by token.
 * A row is
 *   PLAIN  head_dim elements of the call's dtype;
 *   INT4   head_dim / 2 bytes of codes, then for each 32 channels a step and a
 *          low (f16, f16). Of 8 channels in 32 bits, channel 2 n is in bits
 *          4 n .. 4 n + 3, channel 2 n + 1 in bits 16 + 4 n .. A code stands
 *          for the f16 nearest to low + code * step: 5/8 byte a value.
 *
 * table and lengths are device arrays, read when the kernels run. A page
 * number outside the cache is a page that is not there (one given back, or
 * never dealt out): nothing is written to it and its keys are not seen; neither
 * are keys beyond the table's row, of a longer document, whose places count from
 * its whole length all the same. Pages may be shared by documents that read
 * them.
 * ------------------------------------------------------------------------ */
enum { BL_CACHE_PLAIN = 0, BL_CACHE_INT4 = 1 };
#define BL_CACHE_MAX_PAGE_ROWS 256u
#define BL_CACHE_MAX_KEYS (1u << 24) /* of a document: max_pages * page_rows */
#define BL_CACHE_GROUP 32u           /* channels that share a step and a low */

typedef struct {
    void *data;
    uint64_t page_stride, row_stride, head_stride; /* bytes; PLAIN: data and strides are multiples of 16, INT4: of 4 */
} bl_pages;

typedef struct {
    uint32_t kind;           /* BL_CACHE_* */
    uint32_t pages;          /* of the cache */
    uint32_t page_rows;      /* a multiple of 16 up to BL_CACHE_MAX_PAGE_ROWS */
    uint32_t max_pages;      /* of a document: the table's row */
    const int32_t *table;    /* [documents][max_pages] */
    const int32_t *lengths;  /* [documents]: keys of each document, a step's new ones among them */
    bl_pages k, v;
} bl_paged_cache;

/* New keys and values into their documents' pages, with the keys' norm and
 * rotary positions on the way, and the same for the queries beside them.
 *
 * Document d's new rows are [q_offsets[d], q_offsets[d + 1]); with n of them,
 * row i of the document is its key lengths[d] - n + i. A key before the first
 * (n > lengths[d]), beyond the table or of a page that is not there is dropped;
 * its query is turned all the same. Rows of no document are not touched, and
 * of the cache nothing but the new keys' rows. A page's row that two rows of a
 * call are appended to (a page in two documents' tables) may hold parts of both,
 * codes of one under a step and low of the other: a shared page is copied before
 * a document goes on in it.
 *
 * q_out and PLAIN keys are computed in f32 and rounded once; values are copied.
 * INT4: low is the smallest value of a group, step (largest - smallest) / 15,
 * each rounded to f32 and then to f16, and a code the nearest integer to (value
 * - low) / step (ties to even, 0 to 15). Keys are computed in 64 bits for it and
 * rounded to f32, and codes are those of 64 bits: the definition's, whatever
 * alignment the call's tensors have. A group that holds a NaN or a magnitude above 65504
 * stands for NaN. Values up to 65440 in magnitude stand for finite ones: low and
 * step are off by at most 16 and 4, and 65440 + 16 + 15 * 4 is under 65520, where
 * f16 rounds to infinity. With larger ones a group's last code may stand for it. */
typedef struct {
    uint32_t dtype;             /* of q, k, v and a PLAIN cache */
    uint32_t rows;              /* of q, k and v */
    uint32_t documents;
    uint32_t q_heads, kv_heads; /* q_heads 0: no queries */
    uint32_t head_dim;          /* a multiple of 8 (INT4: of 32) up to BL_ATTENTION_MAX_HEAD_DIM */
    uint32_t norm;              /* BL_HEAD_NORM_* */
    float epsilon;
    const int32_t *q_offsets;   /* [documents + 1], not falling; NULL: one document of all rows */
    const int32_t *positions;   /* [rows][axes]; NULL (tables of one axis): each row's key index */
    const void *q_gamma, *k_gamma;
    bl_heads q_in, q_out, k_in, v_in; /* q_out may be q_in itself */
    bl_paged_cache cache;
} bl_cache_append_args;
/* table NULL: no rotation. */
int bl_cache_append(bl_ctx *ctx, const bl_rotary_table *table, const bl_cache_append_args *args);

/* The documents' keys and values from their pages to packed rows, of a PLAIN
 * cache's own type or of any of the three from codes: document d's keys first[d],
 * first[d] + 1 .. to the rows from offsets[d] on, as many as the row ranges and
 * lengths[d] leave. Rows beyond are not touched; those of a page that is not
 * there are zeros. */
typedef struct {
    uint32_t dtype;             /* of k_out and v_out */
    uint32_t rows;              /* of k_out and v_out */
    uint32_t documents;
    uint32_t kv_heads, head_dim;
    const int32_t *offsets;     /* [documents + 1], not falling; NULL: one document of all rows */
    const int32_t *first;       /* [documents]; NULL: zeros */
    bl_heads k_out, v_out;      /* 16-byte aligned, strides multiples of 16 bytes */
    bl_paged_cache cache;
} bl_cache_read_args;
int bl_cache_read(bl_ctx *ctx, const bl_cache_read_args *args);

/* Attention of packed queries over the documents' pages: bl_packed_attention's
 * formulas, without a bias. Document d owns the query rows [q_offsets[d],
 * q_offsets[d + 1]), n of them, and its query i stands at key lengths[d] - n + i
 * (its place), as bl_cache_append put it there.
 *
 *   mask:  NONE every key of the document; CAUSAL keys j <= place, and with a
 *          window only the nearest, j > place - window
 *
 * A row that sees no key gets out = 0 and lse = -inf; rows of no document are
 * not touched. Rows of a page beyond the document's length are never read, and
 * hidden keys, and pages that are not there, may hold anything. A NaN key makes
 * NaN of the rows that see it, infinite and NaN values of their channels (f32
 * over INT4: an infinite key may do as a NaN). Statistics, sums and scores are
 * f32. For the matrix cores probabilities are rounded to the tensors' type over
 * a PLAIN cache (bf16 of few queries a document keeps 15 bits) and to f16 over
 * INT4, where queries are taken times a power of two of each row that keeps them
 * in f16's range; f32 over INT4 takes queries and probabilities as two f16 each.
 * No atomics: equal calls give equal bits. */
typedef struct {
    uint32_t dtype;             /* of q, out and a PLAIN cache */
    uint32_t q_heads, kv_heads; /* q_heads a multiple of kv_heads */
    uint32_t head_dim;          /* a multiple of 8 (INT4: of 32) up to BL_ATTENTION_MAX_HEAD_DIM */
    uint32_t q_rows;
    uint32_t documents;
    uint32_t mask;              /* BL_MASK_NONE or BL_MASK_CAUSAL */
    uint32_t window;            /* 0: all; with BL_MASK_CAUSAL */
    uint32_t max_keys;          /* the longest document's keys as far as the host knows, 0: the table's row. Decides
                                 * how many workgroups share a document; a longer one is computed all the same */
    float scale, softcap;       /* softcap 0: none */
    const int32_t *q_offsets;   /* [documents + 1], not falling; NULL: one document of all rows */
    bl_heads q, out;            /* 16-byte aligned, strides multiples of 16 bytes */
    float *lse;                 /* [q_heads][q_rows] or NULL */
    bl_paged_cache cache;
    void *workspace;            /* 16-byte aligned */
    uint64_t workspace_bytes;
} bl_paged_attention_args;
/* The bytes bl_paged_attention needs with these sizes; pointers are not looked at. */
int bl_paged_attention_workspace(bl_ctx *ctx, const bl_paged_attention_args *args, uint64_t *bytes);
int bl_paged_attention(bl_ctx *ctx, const bl_paged_attention_args *args);

#ifdef __cplusplus
}
#endif
#endif
