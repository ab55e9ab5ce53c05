/*
 * beatlm HIP backend: the operators of an attention sublayer on packed
 * sequences, with their gradients, as direct calls over device pointers:
 * LayerNorm, rotary positions of several axes, and attention over packed
 * documents whose scores may be capped by a tanh and carry a bias that depends
 * on distance, under a document, causal or prefix mask. The reference has no
 * counterpart: it runs one image at a time, forward only, through kernel
 * specs. These calls stand beside bl_flash_attention_static for hosts that
 * train or adapt a model, pack images or videos of several sizes into one
 * batch, or decode tokens over a cache.
 *
 * Conventions are beatlm_hip.h's: every call returns a status (0 ok, negative
 * an error of that header's enum, with bl_last_error's message), launches on
 * the context's stream, allocates nothing and never waits, so it may be
 * captured into a HIP graph by the caller (the argument structs are read
 * during the call alone; device arrays are read when the kernels run). Calls
 * that need scratch take a workspace from the caller, of the size the
 * matching *_workspace call gives; its contents mean nothing between calls.
 * Calls that may overlap in time (two streams, two graphs replayed at once)
 * need a workspace each. The context's device is made current for the call
 * and the caller's current device restored. A refused call launches nothing.
 *
 * A context made by bl_ctx_create has a stream of its own;
 * bl_ctx_create_on makes one over a stream that the host already works on.
 */
#ifndef BEATLM_OPS_H
#define BEATLM_OPS_H

#include <stdint.h>

#include "beatlm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A third element type, of these operators alone (kernel specs refuse it). */
enum { BL_BF16 = 2 };

/* bl_ctx_create over the host's stream (hipStream_t; NULL: the device's
 * default stream): everything the context launches goes there. The host keeps
 * the stream alive as long as the context and what was made from it (arenas,
 * kernels, timers) and orders its own work on it as it likes; destroying the
 * context leaves the stream alone.
 * bl_kernels_encode_range on such a context launches one by one, and the host
 * may capture them into a graph of its own: a replay packs the program's
 * weights again and takes nothing else for held from outside the graph, and
 * after a capture no call takes anything for held from the calls before it.
 * Nothing is timed in a capture. A stream of another device is
 * BL_ERR_INVALID_ARGUMENT. */
int bl_ctx_create_on(int device_ordinal, void *stream, bl_ctx **out);

/* ------------------------------------------------------------------------
 * LayerNorm and its gradients
 *
 *   mean_r = sum_c x[r][c] / cols
 *   rstd_r = 1 / sqrt(sum_c (x[r][c] - mean_r)^2 / cols + epsilon)
 *   n[r][c] = (x[r][c] - mean_r) rstd_r
 *   y[r][c] = n[r][c] gamma[c] + beta[c]
 *
 *   d_beta[c] = sum_r dy[r][c]          d_gamma[c] = sum_r dy[r][c] n[r][c]
 *   dx[r][c] = rstd_r (g - mean_c(g) - n[r][c] mean_c(g n)),  g = dy gamma
 *
 * x, y, dy, dx, gamma and beta have the type `dtype`; the statistics and the
 * weights' gradients are f32, and so is every sum. Rows may be strided; the
 * width is 1 to BL_LAYER_NORM_MAX_COLS. y may be x, and dx may be dy or x
 * (with the same stride); other overlaps of them are refused.
 * rows = 0 writes nothing but zeros to d_gamma and d_beta. The sums over rows
 * are made in a fixed order: equal calls give equal bits.
 * ------------------------------------------------------------------------ */
#define BL_LAYER_NORM_MAX_COLS 16384u
typedef struct {
    uint32_t dtype;              /* BL_F32, BL_F16 or BL_BF16 */
    uint32_t rows, cols;
    float epsilon;               /* >= 0, finite */
    uint64_t x_stride, y_stride; /* elements from a row to the next, >= cols */
    const void *x, *gamma, *beta;
    void *y;                     /* forward only */
    float *mean, *rstd;          /* [rows]; written by the forward unless NULL, read by the backward */
} bl_layer_norm_args;

typedef struct {
    const void *dy;
    uint64_t dy_stride;
    void *dx;
    uint64_t dx_stride;
    float *d_gamma, *d_beta;     /* [cols] */
    void *workspace;             /* 16-byte aligned */
    uint64_t workspace_bytes;
} bl_layer_norm_grads;

int bl_layer_norm(bl_ctx *ctx, const bl_layer_norm_args *args);
int bl_layer_norm_backward_workspace(bl_ctx *ctx, const bl_layer_norm_args *args, uint64_t *bytes);
/* Reads x, gamma, mean and rstd of `args` (y and beta are not used). */
int bl_layer_norm_backward(bl_ctx *ctx, const bl_layer_norm_args *args, const bl_layer_norm_grads *grads);

/* A tensor [rows][heads][head_dim] of element type `dtype`, channels next to
 * each other: element (r, h, c) at data + r * row_stride + h * head_stride + c
 * elements. q, k and v of one projection's output are three such views. */
typedef struct {
    void *data;
    uint64_t row_stride, head_stride;
} bl_heads;

/* ------------------------------------------------------------------------
 * Rotary positions of one to three axes
 *
 * Pair i of a head's channels, (a, b), is turned by the angle
 *   phi = positions[row][axis of i] * frequency of i:
 *   (a cos phi - b sin phi, a sin phi + b cos phi)
 * and channels beyond the pairs are copied. The gradient of a rotation is the
 * rotation by -phi: `inverse` 1 on the gradients. Angles are reduced in 64
 * bits, to within |position| 2^-54 revolutions (less than f32's own step up to
 * positions of 2^28); sines and products are f32.
 * ------------------------------------------------------------------------ */
#define BL_ROTARY_MAX_PAIRS 128u
enum {
    BL_ROTARY_HALVES = 0,    /* pair i is channels i and pairs + i */
    BL_ROTARY_NEIGHBOURS = 1 /* pair i is channels 2 i and 2 i + 1 */
};
enum {
    BL_ROTARY_SHARED = 0,  /* pair i of all pairs: base^(-i / pairs) */
    BL_ROTARY_PER_AXIS = 1 /* pair i of an axis's own section of n: base^(-i / n) */
};
/* Which axis turns each pair and how fast. bl_rotary_table_make fills one; a
 * host with frequencies of its own (stretched ladders, other orders of axes)
 * fills it itself. Passed by value into the launch: nothing to keep alive. */
typedef struct {
    uint32_t axes;    /* 1 to 3 */
    uint32_t pairs;   /* 1 to BL_ROTARY_MAX_PAIRS */
    uint32_t layout;  /* BL_ROTARY_HALVES / _NEIGHBOURS */
    uint32_t reserved;
    double turns[BL_ROTARY_MAX_PAIRS]; /* revolutions per unit of position: frequency / (2 pi) */
    uint8_t axis[BL_ROTARY_MAX_PAIRS];
} bl_rotary_table;

/* sections[a] pairs for axis a, in order (their sum is the table's pairs). No
 * context and no GPU: BL_ERR_INVALID_ARGUMENT when there is nothing to turn,
 * too much, or a base that is not a finite number above 0. */
int bl_rotary_table_make(const uint32_t *sections, uint32_t axes, double base, uint32_t ladder, uint32_t layout,
                         bl_rotary_table *out);

typedef struct {
    uint32_t dtype;
    uint32_t rows;
    uint32_t q_heads, k_heads;  /* either may be 0: that tensor is not touched */
    uint32_t head_dim;          /* 2 * pairs to 256 */
    uint32_t inverse;           /* 0 or 1 */
    const int32_t *positions;   /* [rows][axes] on the device; any int32 */
    bl_heads q_in, q_out, k_in, k_out; /* out may be in itself (the same strides); other overlaps of an output are refused */
} bl_rotary_args;

int bl_rotary(bl_ctx *ctx, const bl_rotary_table *table, const bl_rotary_args *args);

/* ------------------------------------------------------------------------
 * Attention over packed documents, and its gradients
 *
 * Document d owns the query rows [q_offsets[d], q_offsets[d + 1]) and sees the
 * key rows [k_begin[d], k_end[d]), nothing else (the document mask). With n_q
 * queries and n_k keys, its query i stands at the place i + n_k - n_q of its
 * keys, so a packed batch (n_q = n_k), a chunk of a prompt behind a cache and
 * a decoding step (n_q = 1) are one call. Query head h reads key head
 * h / (q_heads / kv_heads).
 *
 *   s = scale * q . k                     softcap > 0: s = softcap * tanh(s / softcap)
 *   slopes: s -= slopes[head] * distance
 *     distance = |i + n_k - n_q - j|, or with positions of `axes` axes
 *                sum_a |q_positions[i][a] - k_positions[j][a]|
 *   mask:  NONE every key of the document; CAUSAL j <= i + n_k - n_q;
 *          PREFIX that, or j < prefix[d]
 *   lse = log sum_j exp(s_j),  out = sum_j exp(s_j - lse) v_j
 *
 * A row that sees no key gets out = 0 and lse = -inf, and no gradient. Rows of
 * no document are not touched, neither in out and lse nor in the gradients;
 * memory outside the documents is never read, so it may hold anything. Hidden
 * scores count as exactly -inf whatever q and k hold there; a hidden key's v
 * may be anything too. Sums, statistics and scores are f32; for the matrix
 * cores the probabilities, and the scores' gradients, are rounded to the
 * tensors' type (f32 stays f32; f16 holds them times powers of two that keep
 * them in its range). What a call writes overlaps nothing else that it
 * touches: tensors that do are refused; lse, d_slopes and the workspace are not
 * looked at.
 *
 * The offsets are device arrays, read when the kernels run (a captured graph
 * may be replayed with others); they are clamped to the tensors' rows, so
 * wrong ones give wrong results but no access outside. `documents` and the
 * tensors' rows are fixed by the call.
 *
 * Gradients (bl_packed_attention_backward): d_q, d_k, d_v with heads of a group summed
 * into their shared key head, and d_slopes summed over rows; fixed order of
 * sums, so equal calls give equal bits. It takes the keys packed by one array
 * of offsets (k_end = k_begin + 1), as documents that shared keys would have
 * to add to each other's gradients. A document whose q, k, v or d_out holds a
 * NaN or an infinity, hidden or not, has gradients that mean nothing, and so
 * do d_slopes of its heads; the other documents' are their own.
 * ------------------------------------------------------------------------ */
#define BL_ATTENTION_MAX_HEAD_DIM 128u
enum { BL_MASK_NONE = 0, BL_MASK_CAUSAL = 1, BL_MASK_PREFIX = 2 };

typedef struct {
    uint32_t dtype;
    uint32_t q_heads, kv_heads; /* q_heads a multiple of kv_heads */
    uint32_t head_dim;          /* a multiple of 8, up to BL_ATTENTION_MAX_HEAD_DIM */
    uint32_t q_rows, k_rows;    /* rows of the tensors */
    uint32_t documents;
    uint32_t mask;              /* BL_MASK_* */
    uint32_t axes;              /* of the positions, 0 to 3; 0: distances are of the tokens' indexes */
    uint32_t max_keys;          /* the longest document's keys as far as the host knows, 0: k_rows. Decides how
                                 * many workgroups share a document; a longer one is computed all the same */
    float scale, softcap;       /* softcap 0: none */
    const int32_t *q_offsets;   /* [documents + 1], not falling; NULL: one document of all rows */
    const int32_t *k_begin, *k_end; /* [documents]; both NULL: one document of all rows */
    const int32_t *prefix;      /* [documents], with BL_MASK_PREFIX */
    const float *slopes;        /* [q_heads] or NULL */
    const int32_t *q_positions, *k_positions; /* [q_rows][axes], [k_rows][axes] when axes > 0, within +-2^28 */
    bl_heads q, k, v;           /* 16-byte aligned, strides multiples of 16 bytes */
    bl_heads out;
    float *lse;                 /* [q_heads][q_rows]; NULL allowed in the forward */
    void *workspace;            /* 16-byte aligned */
    uint64_t workspace_bytes;
} bl_packed_attention_args;

typedef struct {
    bl_heads d_out;
    bl_heads d_q, d_k, d_v;
    float *d_slopes;            /* [q_heads] or NULL */
} bl_packed_attention_grads;

/* The bytes the forward (backward = 0), or the forward and the backward
 * (backward = 1), need with these sizes; pointers are not looked at. */
int bl_packed_attention_workspace(bl_ctx *ctx, const bl_packed_attention_args *args, uint32_t backward, uint64_t *bytes);
int bl_packed_attention(bl_ctx *ctx, const bl_packed_attention_args *args);
/* Reads q, k, v, out and lse of `args` as the forward left them. */
int bl_packed_attention_backward(bl_ctx *ctx, const bl_packed_attention_args *args, const bl_packed_attention_grads *grads);

#ifdef __cplusplus
}
#endif
#endif
