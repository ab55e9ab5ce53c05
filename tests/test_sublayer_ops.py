"""The packed sublayer's operators without a GPU: the header's functions and
struct layouts, the rotary table, and every refusal of their host side, run
as it is (csrc/ops.cpp) over a stand-in for the context and for the launches."""

import ctypes as C
import math
import pathlib
import re
import subprocess

import pytest

from beatlm_amd import hip, ops

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "beatlm_ops.h"


def test_the_library_exports_the_header_s_functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(bl_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 9
    assert [n for n in names if not hasattr(hip.lib(), n)] == []


def test_the_structs_have_the_c_layout(tmp_path):
    structs = {"bl_layer_norm_args": ops.LayerNormArgs, "bl_layer_norm_grads": ops.LayerNormGrads, "bl_heads": ops.Heads,
               "bl_rotary_table": ops.RotaryTable, "bl_rotary_args": ops.RotaryArgs, "bl_packed_attention_args": ops.AttentionArgs,
               "bl_packed_attention_grads": ops.AttentionGrads}
    lines = [f'printf("{n} %zu\\n", sizeof({n}));' for n in structs]
    lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, c in structs.items() for f, *_ in c._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "beatlm_ops.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for key, value in got.items():
        name, _, field = key.partition(".")
        assert int(value) == (getattr(structs[name], field).offset if field else C.sizeof(structs[name])), key
    text = HEADER.read_text()
    for name, value in (("BL_LAYER_NORM_MAX_COLS", ops.LAYER_NORM_MAX_COLS), ("BL_ROTARY_MAX_PAIRS", ops.ROTARY_MAX_PAIRS),
                        ("BL_ATTENTION_MAX_HEAD_DIM", ops.ATTENTION_MAX_HEAD_DIM)):
        assert f"#define {name} {value}u" in text
    assert "BL_BF16 = 2" in text and ops.BF16 == 2


def test_without_a_device_a_context_over_a_stream_is_an_error():
    h = C.c_void_p()
    rc = hip.lib().bl_ctx_create_on(0, None, C.byref(h))
    if rc == hip.OK:
        hip.lib().bl_ctx_destroy(h)
        pytest.skip("a GPU is visible")
    assert rc in (hip.ERR_HIP, hip.ERR_INVALID_ARGUMENT)
    assert hip.lib().bl_ctx_create_on(0, None, None) == hip.ERR_INVALID_ARGUMENT


# ---- the rotary table ----


def test_the_shared_ladder_runs_over_all_pairs():
    t = ops.rotary_table([2, 3, 3], 500.0)
    assert (t.axes, t.pairs, t.layout) == (3, 8, ops.ROTARY_HALVES)
    assert list(t.axis[:8]) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert [t.turns[i] * 2 * math.pi for i in range(8)] == pytest.approx([500.0 ** (-i / 8) for i in range(8)], rel=1e-14)


def test_the_ladder_per_axis_starts_again():
    t = ops.rotary_table([3, 1], 10000.0, per_axis=True, neighbours=True)
    assert t.layout == ops.ROTARY_NEIGHBOURS
    assert [t.turns[i] * 2 * math.pi for i in range(4)] == pytest.approx([1.0, 10000.0 ** (-1 / 3), 10000.0 ** (-2 / 3), 1.0], rel=1e-14)


@pytest.mark.parametrize("sections,base", [([], 10.0), ([0], 10.0), ([0, 0], 10.0), ([129], 10.0), ([1, 1, 1, 1], 10.0), ([4], 0.0), ([4], -2.0),
                                           ([4], math.inf), ([4], math.nan), ([2**32 - 1, 2], 10.0)])
def test_rotary_tables_refused(sections, base):
    with pytest.raises(hip.BackendError) as e:
        ops.rotary_table(sections, base)
    assert e.value.code == hip.ERR_INVALID_ARGUMENT


# ---- refusals: the host side as it is, over stand-ins ----

STAND_INS = r"""
#include <string>
#include "ctx.hpp"
#include "ops.hpp"
struct bl_ctx { std::string error; int launches; };
static bl_ctx the_ctx;
extern "C" bl_ctx *stand_in_ctx() { the_ctx.launches = 0; return &the_ctx; }
extern "C" const char *stand_in_error() { return the_ctx.error.c_str(); }
extern "C" int stand_in_launches() { return the_ctx.launches; }
int bl_fail(bl_ctx *ctx, int code, const char *msg) { ctx->error = msg; return code; }
hipStream_t bl_stream_of(bl_ctx *) { return nullptr; }
int bl_device_of(const bl_ctx *) { return 0; }
uint32_t bl_compute_units_of(const bl_ctx *) { return 256; }
extern "C" hipError_t hipGetDevice(int *d) { *d = 0; return hipSuccess; }
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }
extern "C" const char *hipGetErrorString(hipError_t) { return ""; }
namespace bl {
static hipError_t launch() { the_ctx.launches++; return hipSuccess; }
uint32_t norm_groups(uint32_t rows, uint32_t, uint32_t, uint32_t) { return rows ? 1 : 0; }
hipError_t launch_norm_forward(const NormParams &, uint32_t, hipStream_t) { return launch(); }
hipError_t launch_norm_backward(const NormParams &, uint32_t, hipStream_t) { return launch(); }
hipError_t launch_rotary(const RotaryParams &, uint32_t, uint32_t, hipStream_t) { return launch(); }
PackedPlan plan_packed(const bl_packed_attention_args &, uint32_t) { PackedPlan p{}; p.forward_bytes = 64; p.backward_bytes = 128; return p; }
hipError_t launch_packed_forward(const PackedParams &, const PackedPlan &, hipStream_t) { return launch(); }
hipError_t launch_packed_backward(const PackedParams &, const PackedPlan &, hipStream_t) { return launch(); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("ops")
    (d / "stand_ins.cpp").write_text(STAND_INS)
    csrc = ROOT / "beatlm_amd" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{csrc}",
                    str(csrc / "ops.cpp"), str(d / "stand_ins.cpp"), "-o", str(d / "libops.so"), "-Wl,-Bsymbolic", "-w"], check=True)
    lib = C.CDLL(str(d / "libops.so"))
    lib.stand_in_ctx.restype = C.c_void_p
    lib.stand_in_error.restype = C.c_char_p
    for name, (res, args) in ops._SIG.items():
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


AT = 1 << 20  # an address the stand-ins never look at


def refused(host, call, structs, code, says):
    ctx = host.stand_in_ctx()
    rc = call(ctx, *[C.byref(s) if s is not None else None for s in structs])
    assert rc == code, (rc, host.stand_in_error())
    assert says in host.stand_in_error().decode(), host.stand_in_error()
    assert host.stand_in_launches() == 0


def accepted(host, call, structs, launches=1):
    ctx = host.stand_in_ctx()
    assert call(ctx, *[C.byref(s) for s in structs]) == hip.OK, host.stand_in_error()
    assert host.stand_in_launches() == launches


def norm_args(**changed):
    a = ops.LayerNormArgs(dtype=hip.F16, rows=4, cols=20, epsilon=1e-6, x_stride=20, y_stride=24, x=AT, gamma=AT, beta=AT, y=2 * AT, mean=AT, rstd=AT)
    for name, value in changed.items():
        setattr(a, name, value)
    return a


def norm_grads(**changed):
    g = ops.LayerNormGrads(dy=AT, dy_stride=20, dx=3 * AT, dx_stride=20, d_gamma=AT, d_beta=AT, workspace=AT, workspace_bytes=1 << 20)
    for name, value in changed.items():
        setattr(g, name, value)
    return g


INVALID, LARGE, MISALIGNED = hip.ERR_INVALID_ARGUMENT, hip.ERR_TOO_LARGE, hip.ERR_MISALIGNED_PLACEMENT


@pytest.mark.parametrize("changed,code,says", [
    (dict(dtype=3), INVALID, "dtype"), (dict(cols=0), INVALID, "zero columns"), (dict(cols=16385, x_stride=20000, y_stride=20000), LARGE, "columns"),
    (dict(rows=2**31), LARGE, "rows"), (dict(epsilon=-1.0), INVALID, "epsilon"), (dict(epsilon=math.nan), INVALID, "epsilon"),
    (dict(x_stride=19), INVALID, "x's rows"), (dict(y_stride=0), INVALID, "y's rows"), (dict(x=None), INVALID, "x is null"),
    (dict(y=None), INVALID, "y is null"), (dict(gamma=None), INVALID, "gamma"), (dict(beta=AT + 1), INVALID, "beta is misaligned"),
    (dict(x=AT + 1), INVALID, "x is misaligned"), (dict(mean=AT + 2), INVALID, "statistics"), (dict(y=AT), INVALID, "another stride"),
])
def test_layer_norm_refusals(host, changed, code, says):
    refused(host, host.bl_layer_norm, [norm_args(**changed)], code, says)


@pytest.mark.parametrize("changed,more,code,says", [
    ({}, dict(dy=None), INVALID, "dy is null"), ({}, dict(dx=None), INVALID, "dx is null"), ({}, dict(dx_stride=3), INVALID, "dx's rows"),
    ({}, dict(d_gamma=None), INVALID, "d_gamma"), ({}, dict(d_beta=AT + 2), INVALID, "d_beta"), (dict(mean=None), {}, INVALID, "mean"),
    (dict(rstd=None), {}, INVALID, "rstd"), ({}, dict(workspace_bytes=8), LARGE, "workspace"), ({}, dict(workspace=None), MISALIGNED, "workspace"),
    ({}, dict(workspace=AT + 4), MISALIGNED, "workspace"), (dict(x_stride=28), dict(dx=AT), INVALID, "another stride"), (dict(cols=0), {}, INVALID, "zero"),
])
def test_layer_norm_backward_refusals(host, changed, more, code, says):
    refused(host, host.bl_layer_norm_backward, [norm_args(**changed), norm_grads(**more)], code, says)


def test_layer_norm_accepted(host):
    accepted(host, host.bl_layer_norm, [norm_args()])
    accepted(host, host.bl_layer_norm, [norm_args(rows=0, x=None, y=None)], 0)
    accepted(host, host.bl_layer_norm_backward, [norm_args(y=None, beta=None), norm_grads()])
    accepted(host, host.bl_layer_norm_backward, [norm_args(rows=0, x=None, mean=None, rstd=None), norm_grads(dy=None, dx=None, workspace=None, workspace_bytes=0)])
    refused(host, host.bl_layer_norm, [None], INVALID, "no arguments")
    refused(host, host.bl_layer_norm_backward, [norm_args(), None], INVALID, "no gradients")
    assert host.bl_layer_norm(None, C.byref(norm_args())) == INVALID


def rotary_args(**changed):
    v = ops.Heads(AT, 256, 64)
    a = ops.RotaryArgs(dtype=hip.F32, rows=9, q_heads=4, k_heads=2, head_dim=64, positions=AT, q_in=v, q_out=ops.Heads(2 * AT, 256, 64), k_in=v,
                       k_out=ops.Heads(3 * AT, 256, 64))
    for name, value in changed.items():
        setattr(a, name, value)
    return a


def table(**changed):
    t = ops.rotary_table([16, 16], 100.0)
    for name, value in changed.items():
        setattr(t, name, value)
    return t


def table_with(pair, axis=0, turns=0.1):
    t = table()
    t.axis[pair], t.turns[pair] = axis, turns
    return t


@pytest.mark.parametrize("t,changed,code,says", [
    (table(), dict(dtype=9), INVALID, "dtype"), (table(axes=0), {}, INVALID, "table"), (table(axes=4), {}, INVALID, "table"), (table(pairs=0), {}, INVALID, "table"),
    (table(pairs=129), {}, INVALID, "table"), (table(layout=2), {}, INVALID, "table"), (table_with(5, axis=2), {}, INVALID, "pair 5"),
    (table_with(31, turns=math.nan), {}, INVALID, "pair 31"), (table(), dict(head_dim=63), INVALID, "heads of 63"), (table(), dict(head_dim=257), INVALID, "heads"),
    (table(), dict(inverse=2), INVALID, "inverse"), (table(), dict(q_heads=0, k_heads=0), INVALID, "no heads"), (table(), dict(rows=2**31), LARGE, "rows"),
    (table(), dict(positions=None), INVALID, "positions"), (table(), dict(positions=AT + 2), INVALID, "positions"),
    (table(), dict(q_in=ops.Heads(None, 256, 64)), INVALID, "q_in is null"), (table(), dict(k_out=ops.Heads(AT + 2, 256, 64)), MISALIGNED, "k_out"),
    (table(), dict(q_out=ops.Heads(AT, 128, 64)), INVALID, "other strides"), (table(), dict(k_out=ops.Heads(2 * AT, 256, 32)), INVALID, "overlap"),
    (table(), dict(k_out=ops.Heads(2 * AT, 60, 64)), INVALID, "overlap"), (table(), dict(q_in=ops.Heads(AT, 2**40, 64)), LARGE, "strides"),
])
def test_rotary_refusals(host, t, changed, code, says):
    refused(host, host.bl_rotary, [t, rotary_args(**changed)], code, says)


def test_rotary_accepted(host):
    accepted(host, host.bl_rotary, [table(), rotary_args()])
    accepted(host, host.bl_rotary, [table(), rotary_args(rows=0, positions=None)], 0)
    accepted(host, host.bl_rotary, [table(), rotary_args(k_heads=0, k_in=ops.Heads(), k_out=ops.Heads())])
    accepted(host, host.bl_rotary, [table(), rotary_args(q_out=ops.Heads(AT, 256, 64))])


def attention_args(**changed):
    v = ops.Heads(AT, 256, 64)
    a = ops.AttentionArgs(dtype=ops.BF16, q_heads=4, kv_heads=2, head_dim=64, q_rows=10, k_rows=20, documents=2, scale=0.125, q_offsets=AT, k_begin=AT, k_end=AT + 4,
                          q=v, k=v, v=v, out=ops.Heads(2 * AT, 256, 64), lse=AT, workspace=AT, workspace_bytes=4096)
    for name, value in changed.items():
        setattr(a, name, value)
    return a


def attention_grads(**changed):
    g = ops.AttentionGrads(d_out=ops.Heads(AT, 256, 64), d_q=ops.Heads(5 * AT, 256, 64), d_k=ops.Heads(3 * AT, 128, 64), d_v=ops.Heads(4 * AT, 128, 64))
    for name, value in changed.items():
        setattr(g, name, value)
    return g


ATTENTION_REFUSALS = [
    (dict(dtype=3), INVALID, "dtype"), (dict(q_heads=3), INVALID, "3 query heads over 2"), (dict(kv_heads=0), INVALID, "heads"), (dict(q_heads=0), INVALID, "heads"),
    (dict(head_dim=60), INVALID, "heads of 60"), (dict(head_dim=0), INVALID, "heads of 0"), (dict(head_dim=136), LARGE, "heads of 136"),
    (dict(documents=0), INVALID, "documents"), (dict(documents=2**25), LARGE, "documents"), (dict(mask=3), INVALID, "mask"), (dict(axes=4), INVALID, "axes"),
    (dict(scale=math.inf), INVALID, "scale"), (dict(softcap=-1.0), INVALID, "softcap"), (dict(softcap=math.nan), INVALID, "softcap"),
    (dict(q_rows=2**31), LARGE, "rows"), (dict(k_rows=2**31), LARGE, "rows"), (dict(k_end=None), INVALID, "k_end"), (dict(q_offsets=None), INVALID, "without offsets"),
    (dict(k_begin=None, k_end=None), INVALID, "without offsets"), (dict(mask=2), INVALID, "prefix"), (dict(axes=1), INVALID, "positions without slopes"),
    (dict(axes=1, slopes=AT), INVALID, "without positions"), (dict(axes=2, slopes=AT, q_positions=AT), INVALID, "without positions"),
    (dict(q_offsets=AT + 2), MISALIGNED, "32-bit"), (dict(lse=AT + 1), MISALIGNED, "32-bit"),
    (dict(q=ops.Heads(None, 256, 64)), INVALID, "q is null"), (dict(k=ops.Heads(AT + 8, 256, 64)), MISALIGNED, "k's"), (dict(v=ops.Heads(AT, 252, 64)), MISALIGNED, "v's"),
    (dict(v=ops.Heads(AT, 256, 68)), MISALIGNED, "v's"), (dict(out=ops.Heads(AT, 256, 32)), INVALID, "overlap"), (dict(k=ops.Heads(AT, 2**24, 64)), LARGE, "strides"),
    (dict(workspace_bytes=8), LARGE, "workspace"), (dict(workspace=None), MISALIGNED, "workspace"), (dict(workspace=AT + 8), MISALIGNED, "workspace"),
]


@pytest.mark.parametrize("changed,code,says", ATTENTION_REFUSALS)
def test_attention_refusals(host, changed, code, says):
    refused(host, host.bl_packed_attention, [attention_args(**changed)], code, says)
    refused(host, host.bl_packed_attention_backward, [attention_args(**changed), attention_grads()], code, says)


@pytest.mark.parametrize("changed,more,code,says", [
    (dict(k_end=AT + 400), {}, INVALID, "packed"), (dict(lse=None), {}, INVALID, "lse"), ({}, dict(d_slopes=AT), INVALID, "slopes"),
    (dict(slopes=AT), dict(d_slopes=AT + 2), INVALID, "slopes"), ({}, dict(d_out=ops.Heads()), INVALID, "d_out is null"), ({}, dict(d_q=ops.Heads(AT + 2, 256, 64)), MISALIGNED, "d_q"),
    ({}, dict(d_k=ops.Heads(AT, 128, 0)), INVALID, "d_k's heads"), ({}, dict(d_v=ops.Heads(AT, 0, 64)), INVALID, "d_v's heads"), (dict(workspace_bytes=100), {}, LARGE, "128 are needed"),
])
def test_attention_backward_refusals(host, changed, more, code, says):
    refused(host, host.bl_packed_attention_backward, [attention_args(**changed), attention_grads(**more)], code, says)


def test_attention_accepted(host):
    accepted(host, host.bl_packed_attention, [attention_args()])
    accepted(host, host.bl_packed_attention, [attention_args(lse=None, k=ops.Heads(AT, 0, 0))])
    accepted(host, host.bl_packed_attention, [attention_args(q_rows=0, q=ops.Heads(), out=ops.Heads())], 0)
    accepted(host, host.bl_packed_attention, [attention_args(documents=1, q_offsets=None, k_begin=None, k_end=None)])
    accepted(host, host.bl_packed_attention_backward, [attention_args(slopes=AT), attention_grads(d_slopes=AT)])
    refused(host, host.bl_packed_attention_backward, [attention_args(), None], INVALID, "no gradients")
    n = C.c_uint64()
    ctx = host.stand_in_ctx()
    assert host.bl_packed_attention_workspace(ctx, C.byref(ops.AttentionArgs(dtype=hip.F16, q_heads=1, kv_heads=1, head_dim=8, documents=1)), 1, C.byref(n)) == hip.OK
    assert n.value == 128
    assert host.bl_packed_attention_workspace(ctx, C.byref(attention_args()), 2, C.byref(n)) == INVALID
    assert host.bl_packed_attention_workspace(ctx, C.byref(attention_args()), 0, None) == INVALID


@pytest.mark.parametrize("changed,code,says", [
    (dict(scale=3e38), INVALID, "beyond f32"), (dict(softcap=3e38), INVALID, "beyond f32"), (dict(softcap=1e-40), INVALID, "beyond f32"),
    (dict(out=ops.Heads(AT, 256, 64)), INVALID, "out is q"), (dict(k=ops.Heads(2 * AT, 256, 64)), INVALID, "out is k"), (dict(out=ops.Heads(2 * AT, 64, 64)), INVALID, "overlap"),
    (dict(out=ops.Heads(2 * AT, 248, 64)), INVALID, "overlap"), (dict(out=ops.Heads(2 * AT, 64, 632)), INVALID, "overlap"),
    (dict(k_rows=2**29), LARGE, "rows"), (dict(documents=2**23), LARGE, "documents"),
])
def test_attention_refuses_what_it_would_write_twice_or_could_not_launch(host, changed, code, says):
    refused(host, host.bl_packed_attention, [attention_args(**changed)], code, says)


@pytest.mark.parametrize("more,says", [
    (dict(d_q=ops.Heads(AT, 256, 64)), "d_q is q"), (dict(d_v=ops.Heads(3 * AT, 128, 64)), "d_v is d_k"), (dict(d_k=ops.Heads(5 * AT, 256, 64)), "d_k is d_q"),
    (dict(d_out=ops.Heads(4 * AT, 256, 64)), "d_v is d_out"), (dict(d_q=ops.Heads(2 * AT, 256, 64)), "d_q is out"),
])
def test_gradients_of_attention_lie_apart(host, more, says):
    refused(host, host.bl_packed_attention_backward, [attention_args(), attention_grads(**more)], INVALID, says)


def test_attention_takes_heads_and_rows_in_either_order(host):
    accepted(host, host.bl_packed_attention, [attention_args(out=ops.Heads(2 * AT, 64, 640))])
    accepted(host, host.bl_packed_attention, [attention_args(q_rows=1, out=ops.Heads(2 * AT, 0, 64))])
    accepted(host, host.bl_packed_attention, [attention_args(k_rows=0, k=ops.Heads(2 * AT, 0, 0))])
    accepted(host, host.bl_packed_attention, [attention_args(softcap=1e-30)])
