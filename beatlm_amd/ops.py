"""ctypes binding of the packed attention sublayer's operators
(include/beatlm_ops.h): LayerNorm, rotary positions of several axes and
attention over packed documents, with their gradients; and of those beside them
(include/beatlm_cache.h): norms of each head with its rotary positions, and a
cache of keys in pages, what appends to it, reads it back and attends over it.

The argument structs hold device addresses (an arena's `device_ptr`, another
library's buffer) and are read during the call alone, so a program keeps one
beside its buffers and calls with it again. Nothing here allocates device
memory or waits; the calls run on the context's stream (`hip.Context(device,
stream=...)` for a host that has one already).
"""

from __future__ import annotations

import ctypes as C

from .hip import Context, BackendError, OK, lib

BF16 = 2  # beside hip.F32 and hip.F16, in these operators alone

LAYER_NORM_MAX_COLS = 16384
ROTARY_MAX_PAIRS = 128
ATTENTION_MAX_HEAD_DIM = 128
HEAD_NORM_MAX_HEAD_DIM = 256
CACHE_MAX_PAGE_ROWS = 256
CACHE_MAX_KEYS = 1 << 24
CACHE_GROUP = 32

ROTARY_HALVES, ROTARY_NEIGHBOURS = 0, 1
ROTARY_SHARED, ROTARY_PER_AXIS = 0, 1
MASK_NONE, MASK_CAUSAL, MASK_PREFIX = 0, 1, 2
HEAD_NORM_NONE, HEAD_NORM_RMS, HEAD_NORM_CENTRED = 0, 1, 2
CACHE_PLAIN, CACHE_INT4 = 0, 1

_U32, _U64, _F32, _P = C.c_uint32, C.c_uint64, C.c_float, C.c_void_p


class LayerNormArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("rows", _U32), ("cols", _U32), ("epsilon", _F32),
        ("x_stride", _U64), ("y_stride", _U64),
        ("x", _P), ("gamma", _P), ("beta", _P), ("y", _P), ("mean", _P), ("rstd", _P),
    ]


class LayerNormGrads(C.Structure):
    _fields_ = [
        ("dy", _P), ("dy_stride", _U64), ("dx", _P), ("dx_stride", _U64),
        ("d_gamma", _P), ("d_beta", _P), ("workspace", _P), ("workspace_bytes", _U64),
    ]


class Heads(C.Structure):
    """[rows][heads][head_dim] at a device address; strides in elements."""

    _fields_ = [("data", _P), ("row_stride", _U64), ("head_stride", _U64)]


class RotaryTable(C.Structure):
    _fields_ = [
        ("axes", _U32), ("pairs", _U32), ("layout", _U32), ("reserved", _U32),
        ("turns", C.c_double * ROTARY_MAX_PAIRS), ("axis", C.c_uint8 * ROTARY_MAX_PAIRS),
    ]


class RotaryArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("rows", _U32), ("q_heads", _U32), ("k_heads", _U32), ("head_dim", _U32), ("inverse", _U32),
        ("positions", _P), ("q_in", Heads), ("q_out", Heads), ("k_in", Heads), ("k_out", Heads),
    ]


class AttentionArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("q_heads", _U32), ("kv_heads", _U32), ("head_dim", _U32), ("q_rows", _U32), ("k_rows", _U32),
        ("documents", _U32), ("mask", _U32), ("axes", _U32), ("max_keys", _U32), ("scale", _F32), ("softcap", _F32),
        ("q_offsets", _P), ("k_begin", _P), ("k_end", _P), ("prefix", _P), ("slopes", _P),
        ("q_positions", _P), ("k_positions", _P),
        ("q", Heads), ("k", Heads), ("v", Heads), ("out", Heads), ("lse", _P), ("workspace", _P), ("workspace_bytes", _U64),
    ]


class AttentionGrads(C.Structure):
    _fields_ = [("d_out", Heads), ("d_q", Heads), ("d_k", Heads), ("d_v", Heads), ("d_slopes", _P)]


class HeadNormArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("rows", _U32), ("q_heads", _U32), ("k_heads", _U32), ("head_dim", _U32), ("norm", _U32), ("epsilon", _F32),
        ("positions", _P), ("q_gamma", _P), ("k_gamma", _P), ("q_in", Heads), ("q_out", Heads), ("k_in", Heads), ("k_out", Heads),
    ]


class HeadNormGrads(C.Structure):
    _fields_ = [
        ("dq_out", Heads), ("dk_out", Heads), ("dq_in", Heads), ("dk_in", Heads),
        ("d_q_gamma", _P), ("d_k_gamma", _P), ("workspace", _P), ("workspace_bytes", _U64),
    ]


class Pages(C.Structure):
    """Rows of (page, row, head) at a device address; strides in bytes."""

    _fields_ = [("data", _P), ("page_stride", _U64), ("row_stride", _U64), ("head_stride", _U64)]


class PagedCache(C.Structure):
    _fields_ = [
        ("kind", _U32), ("pages", _U32), ("page_rows", _U32), ("max_pages", _U32), ("table", _P), ("lengths", _P), ("k", Pages), ("v", Pages),
    ]


class CacheAppendArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("rows", _U32), ("documents", _U32), ("q_heads", _U32), ("kv_heads", _U32), ("head_dim", _U32), ("norm", _U32), ("epsilon", _F32),
        ("q_offsets", _P), ("positions", _P), ("q_gamma", _P), ("k_gamma", _P),
        ("q_in", Heads), ("q_out", Heads), ("k_in", Heads), ("v_in", Heads), ("cache", PagedCache),
    ]


class CacheReadArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("rows", _U32), ("documents", _U32), ("kv_heads", _U32), ("head_dim", _U32),
        ("offsets", _P), ("first", _P), ("k_out", Heads), ("v_out", Heads), ("cache", PagedCache),
    ]


class PagedAttentionArgs(C.Structure):
    _fields_ = [
        ("dtype", _U32), ("q_heads", _U32), ("kv_heads", _U32), ("head_dim", _U32), ("q_rows", _U32), ("documents", _U32),
        ("mask", _U32), ("window", _U32), ("max_keys", _U32), ("scale", _F32), ("softcap", _F32),
        ("q_offsets", _P), ("q", Heads), ("out", Heads), ("lse", _P), ("cache", PagedCache), ("workspace", _P), ("workspace_bytes", _U64),
    ]


_SIG = {
    "bl_layer_norm": (C.c_int, [_P, C.POINTER(LayerNormArgs)]),
    "bl_layer_norm_backward_workspace": (C.c_int, [_P, C.POINTER(LayerNormArgs), C.POINTER(_U64)]),
    "bl_layer_norm_backward": (C.c_int, [_P, C.POINTER(LayerNormArgs), C.POINTER(LayerNormGrads)]),
    "bl_rotary_table_make": (C.c_int, [C.POINTER(_U32), _U32, C.c_double, _U32, _U32, C.POINTER(RotaryTable)]),
    "bl_rotary": (C.c_int, [_P, C.POINTER(RotaryTable), C.POINTER(RotaryArgs)]),
    "bl_packed_attention_workspace": (C.c_int, [_P, C.POINTER(AttentionArgs), _U32, C.POINTER(_U64)]),
    "bl_packed_attention": (C.c_int, [_P, C.POINTER(AttentionArgs)]),
    "bl_packed_attention_backward": (C.c_int, [_P, C.POINTER(AttentionArgs), C.POINTER(AttentionGrads)]),
}
# include/beatlm_cache.h
_CACHE_SIG = {
    "bl_head_norm_rotary": (C.c_int, [_P, C.POINTER(RotaryTable), C.POINTER(HeadNormArgs)]),
    "bl_head_norm_rotary_backward_workspace": (C.c_int, [_P, C.POINTER(HeadNormArgs), C.POINTER(_U64)]),
    "bl_head_norm_rotary_backward": (C.c_int, [_P, C.POINTER(RotaryTable), C.POINTER(HeadNormArgs), C.POINTER(HeadNormGrads)]),
    "bl_cache_append": (C.c_int, [_P, C.POINTER(RotaryTable), C.POINTER(CacheAppendArgs)]),
    "bl_cache_read": (C.c_int, [_P, C.POINTER(CacheReadArgs)]),
    "bl_paged_attention_workspace": (C.c_int, [_P, C.POINTER(PagedAttentionArgs), C.POINTER(_U64)]),
    "bl_paged_attention": (C.c_int, [_P, C.POINTER(PagedAttentionArgs)]),
}
_bound = None


def _lib():
    global _bound
    if _bound is None:
        h = lib()
        for name, (res, args) in {**_SIG, **_CACHE_SIG}.items():
            fn = getattr(h, name)
            fn.restype = res
            fn.argtypes = args
        _bound = h
    return _bound


def layer_norm(ctx: Context, args: LayerNormArgs) -> None:
    ctx.check(_lib().bl_layer_norm(ctx.handle, C.byref(args)))


def layer_norm_backward_workspace(ctx: Context, args: LayerNormArgs) -> int:
    """Bytes of the workspace layer_norm_backward needs for these sizes."""
    n = _U64()
    ctx.check(_lib().bl_layer_norm_backward_workspace(ctx.handle, C.byref(args), C.byref(n)))
    return int(n.value)


def layer_norm_backward(ctx: Context, args: LayerNormArgs, grads: LayerNormGrads) -> None:
    ctx.check(_lib().bl_layer_norm_backward(ctx.handle, C.byref(args), C.byref(grads)))


def rotary_table(sections, base: float, per_axis: bool = False, neighbours: bool = False) -> RotaryTable:
    """Which axis turns each pair and how fast: `sections[a]` pairs for axis a,
    frequencies base^(-i / n) over all pairs, or with `per_axis` over each
    section; a pair is channels (i, pairs + i), or with `neighbours`
    (2 i, 2 i + 1). No context, no GPU."""
    t = RotaryTable()
    arr = (_U32 * max(1, len(sections)))(*sections)
    rc = _lib().bl_rotary_table_make(arr, len(sections), base, ROTARY_PER_AXIS if per_axis else ROTARY_SHARED,
                                     ROTARY_NEIGHBOURS if neighbours else ROTARY_HALVES, C.byref(t))
    if rc != OK:
        raise BackendError(rc, f"no rotary table of sections {list(sections)} and base {base}")
    return t


def rotary(ctx: Context, table: RotaryTable, args: RotaryArgs) -> None:
    ctx.check(_lib().bl_rotary(ctx.handle, C.byref(table), C.byref(args)))


def attention_workspace(ctx: Context, args: AttentionArgs, backward: bool = False) -> int:
    """Bytes of the workspace attention, or attention and attention_backward,
    need for these sizes."""
    n = _U64()
    ctx.check(_lib().bl_packed_attention_workspace(ctx.handle, C.byref(args), 1 if backward else 0, C.byref(n)))
    return int(n.value)


def attention(ctx: Context, args: AttentionArgs) -> None:
    ctx.check(_lib().bl_packed_attention(ctx.handle, C.byref(args)))


def attention_backward(ctx: Context, args: AttentionArgs, grads: AttentionGrads) -> None:
    ctx.check(_lib().bl_packed_attention_backward(ctx.handle, C.byref(args), C.byref(grads)))


def _table(table: RotaryTable | None):
    return None if table is None else C.byref(table)


def head_norm_rotary(ctx: Context, table: RotaryTable | None, args: HeadNormArgs) -> None:
    """table None: norms alone."""
    ctx.check(_lib().bl_head_norm_rotary(ctx.handle, _table(table), C.byref(args)))


def head_norm_rotary_backward_workspace(ctx: Context, args: HeadNormArgs) -> int:
    """Bytes of the workspace head_norm_rotary_backward needs for these sizes."""
    n = _U64()
    ctx.check(_lib().bl_head_norm_rotary_backward_workspace(ctx.handle, C.byref(args), C.byref(n)))
    return int(n.value)


def head_norm_rotary_backward(ctx: Context, table: RotaryTable | None, args: HeadNormArgs, grads: HeadNormGrads) -> None:
    ctx.check(_lib().bl_head_norm_rotary_backward(ctx.handle, _table(table), C.byref(args), C.byref(grads)))


def cache_append(ctx: Context, table: RotaryTable | None, args: CacheAppendArgs) -> None:
    """table None: no rotation."""
    ctx.check(_lib().bl_cache_append(ctx.handle, _table(table), C.byref(args)))


def cache_read(ctx: Context, args: CacheReadArgs) -> None:
    ctx.check(_lib().bl_cache_read(ctx.handle, C.byref(args)))


def paged_attention_workspace(ctx: Context, args: PagedAttentionArgs) -> int:
    """Bytes of the workspace paged_attention needs for these sizes."""
    n = _U64()
    ctx.check(_lib().bl_paged_attention_workspace(ctx.handle, C.byref(args), C.byref(n)))
    return int(n.value)


def paged_attention(ctx: Context, args: PagedAttentionArgs) -> None:
    ctx.check(_lib().bl_paged_attention(ctx.handle, C.byref(args)))
