"""ctypes binding of the packed attention sublayer's operators
(include/beatlm_ops.h): LayerNorm, rotary positions of several axes and
attention over packed documents, with their gradients.

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

ROTARY_HALVES, ROTARY_NEIGHBOURS = 0, 1
ROTARY_SHARED, ROTARY_PER_AXIS = 0, 1
MASK_NONE, MASK_CAUSAL, MASK_PREFIX = 0, 1, 2

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
_bound = None


def _lib():
    global _bound
    if _bound is None:
        h = lib()
        for name, (res, args) in _SIG.items():
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
