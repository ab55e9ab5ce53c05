"""The norms of heads and the cache of pages without a GPU: the header's
functions and struct layouts, every refusal of their host side, run as it is
(csrc/cache_ops.cpp) over a stand-in for the context and for the launches, and
what the calls make of the HIP runtime's answers."""

import ctypes as C
import math
import pathlib
import re
import subprocess

import pytest

from beatlm_amd import hip, ops
from tests.test_sublayer_errors import run  # noqa: F401
from tests.test_sublayer_ops import STAND_INS

ROOT = pathlib.Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "beatlm_cache.h"
STRUCTS = {"bl_head_norm_args": ops.HeadNormArgs, "bl_head_norm_grads": ops.HeadNormGrads, "bl_pages": ops.Pages, "bl_paged_cache": ops.PagedCache,
           "bl_cache_append_args": ops.CacheAppendArgs, "bl_cache_read_args": ops.CacheReadArgs, "bl_paged_attention_args": ops.PagedAttentionArgs}


def test_the_library_exports_the_header_s_functions():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = sorted(set(re.findall(r"\b(bl_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(ops._CACHE_SIG)
    assert [n for n in names if not hasattr(hip.lib(), n)] == []


def test_the_structs_have_the_c_layout(tmp_path):
    lines = [f'printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS]
    lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, c in STRUCTS.items() for f, *_ in c._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "beatlm_cache.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.rsplit(" ", 1) for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for key, value in got.items():
        name, _, field = key.partition(".")
        assert int(value) == (getattr(STRUCTS[name], field).offset if field else C.sizeof(STRUCTS[name])), key
    text = HEADER.read_text()
    for line in (f"BL_HEAD_NORM_MAX_HEAD_DIM {ops.HEAD_NORM_MAX_HEAD_DIM}u", f"BL_CACHE_MAX_PAGE_ROWS {ops.CACHE_MAX_PAGE_ROWS}u", f"BL_CACHE_GROUP {ops.CACHE_GROUP}u",
                 "BL_CACHE_MAX_KEYS (1u << 24)"):
        assert f"#define {line}" in text
    assert ops.CACHE_MAX_KEYS == 1 << 24
    assert "BL_HEAD_NORM_NONE = 0, BL_HEAD_NORM_RMS = 1, BL_HEAD_NORM_CENTRED = 2" in text and "BL_CACHE_PLAIN = 0, BL_CACHE_INT4 = 1" in text


# ---- refusals ----

MORE = r"""
namespace bl {
hipError_t launch_heads_forward(const HeadsParams &, uint32_t, uint32_t, hipStream_t) { return launch(); }
hipError_t launch_heads_backward(const HeadsParams &, uint32_t, uint32_t, hipStream_t) { return launch(); }
hipError_t launch_cache_append(const AppendParams &, uint32_t, uint32_t, hipStream_t) { return launch(); }
hipError_t launch_cache_read(const bl_cache_read_args &, uint32_t, hipStream_t) { return launch(); }
template <> hipError_t paged_attention<float>(const PagedParams &, const PagedPlan &, hipStream_t) { return launch(); }
template <> hipError_t paged_attention<_Float16>(const PagedParams &, const PagedPlan &, hipStream_t) { return launch(); }
template <> hipError_t paged_attention<__bf16>(const PagedParams &, const PagedPlan &, hipStream_t) { return launch(); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("cache")
    (d / "stand_ins.cpp").write_text(STAND_INS + MORE)
    csrc = ROOT / "beatlm_amd" / "csrc"
    subprocess.run(["/opt/rocm/llvm/bin/clang++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{csrc}",
                    str(csrc / "cache_ops.cpp"), str(csrc / "paged_plan.cpp"), str(d / "stand_ins.cpp"), "-o", str(d / "libcache.so"), "-Wl,-Bsymbolic", "-w"],
                   check=True)
    lib = C.CDLL(str(d / "libcache.so"))
    lib.stand_in_ctx.restype = C.c_void_p
    lib.stand_in_error.restype = C.c_char_p
    for name, (res, args) in ops._CACHE_SIG.items():
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


AT = 1 << 30  # addresses that the stand-ins never look at
INVALID, LARGE, MISALIGNED = hip.ERR_INVALID_ARGUMENT, hip.ERR_TOO_LARGE, hip.ERR_MISALIGNED_PLACEMENT


def call(host, name, *structs):
    ctx = host.stand_in_ctx()
    rc = getattr(host, name)(ctx, *[C.byref(s) if s is not None else None for s in structs])
    return rc, host.stand_in_error().decode(), host.stand_in_launches()


def refused(host, name, structs, code, says):
    rc, message, launches = call(host, name, *structs)
    assert (rc, launches) == (code, 0) and says in message, (rc, message, launches)


def accepted(host, name, structs, launches=1):
    assert call(host, name, *structs)[::2] == (hip.OK, launches), call(host, name, *structs)


def with_(struct, changed):
    for name, value in changed.items():
        *path, last = name.split("__")
        target = struct
        for p in path:
            target = getattr(target, p)
        setattr(target, last, value)
    return struct


def view(n, heads=4):
    return ops.Heads(n * AT, heads * 64, 64)


def table():
    return ops.rotary_table([16], 100.0)


def norm_args(**changed):
    return with_(ops.HeadNormArgs(dtype=hip.F16, rows=9, q_heads=4, k_heads=2, head_dim=64, norm=ops.HEAD_NORM_RMS, epsilon=1e-6, positions=AT, q_gamma=AT,
                                  k_gamma=AT, q_in=view(2), q_out=view(3), k_in=view(4, 2), k_out=view(5, 2)), changed)


def norm_grads(**changed):
    return with_(ops.HeadNormGrads(dq_out=view(6), dk_out=view(7, 2), dq_in=view(8), dk_in=view(9, 2), d_q_gamma=AT, d_k_gamma=AT, workspace=AT,
                                   workspace_bytes=1 << 20), changed)


def cache(kind=ops.CACHE_PLAIN, **changed):
    row = 40 if kind == ops.CACHE_INT4 else 128
    pages = lambda n: ops.Pages(n * AT, 2 * 16 * row, row, 16 * row)  # noqa: E731
    return with_(ops.PagedCache(kind=kind, pages=10, page_rows=16, max_pages=5, table=AT, lengths=AT, k=pages(20), v=pages(21)), changed)


def append_args(kind=ops.CACHE_PLAIN, **changed):
    return with_(ops.CacheAppendArgs(dtype=hip.F16, rows=9, documents=3, q_heads=4, kv_heads=2, head_dim=64, norm=ops.HEAD_NORM_RMS, epsilon=1e-6, q_offsets=AT,
                                     q_gamma=AT, k_gamma=AT, q_in=view(2), q_out=view(3), k_in=view(4, 2), v_in=view(5, 2), cache=cache(kind)), changed)


def read_args(kind=ops.CACHE_PLAIN, **changed):
    return with_(ops.CacheReadArgs(dtype=hip.F16, rows=9, documents=3, kv_heads=2, head_dim=64, offsets=AT, k_out=view(4, 2), v_out=view(5, 2), cache=cache(kind)), changed)


def attention_args(kind=ops.CACHE_PLAIN, **changed):
    return with_(ops.PagedAttentionArgs(dtype=hip.F16, q_heads=4, kv_heads=2, head_dim=64, q_rows=9, documents=3, mask=ops.MASK_CAUSAL, scale=0.125, q_offsets=AT,
                                        q=view(2), out=view(3), lse=AT, cache=cache(kind), workspace=AT, workspace_bytes=1 << 30), changed)


NORM_REFUSALS = [
    (dict(dtype=3), INVALID, "dtype"), (dict(head_dim=0), INVALID, "no channels"), (dict(head_dim=257), LARGE, "heads of 257"), (dict(norm=0), INVALID, "norm 0"),
    (dict(norm=3), INVALID, "norm 3"), (dict(epsilon=-1.0), INVALID, "epsilon"), (dict(epsilon=math.inf), INVALID, "epsilon"),
    (dict(q_heads=0, k_heads=0), INVALID, "no heads"), (dict(rows=2**31), LARGE, "rows"), (dict(q_heads=70000), LARGE, "heads"),
    (dict(positions=None), INVALID, "positions"), (dict(positions=AT + 2), INVALID, "positions"), (dict(head_dim=31), INVALID, "16 pairs"),
    (dict(q_gamma=AT + 1), MISALIGNED, "q_gamma"), (dict(k_gamma=AT + 1), MISALIGNED, "k_gamma"), (dict(q_in=ops.Heads(None, 256, 64)), INVALID, "q_in is null"),
    (dict(k_in=ops.Heads(4 * AT + 1, 128, 64)), MISALIGNED, "k_in"), (dict(q_in=ops.Heads(2 * AT, 1 << 25, 64)), LARGE, "strides"),
]


@pytest.mark.parametrize("changed,code,says", NORM_REFUSALS + [
    (dict(q_out=ops.Heads(2 * AT, 512, 64)), INVALID, "other strides"), (dict(q_out=ops.Heads(2 * AT + 128, 256, 64)), INVALID, "overlaps q_in"),
    (dict(q_out=ops.Heads(3 * AT, 256, 32)), INVALID, "overlap"), (dict(k_out=view(3, 2)), INVALID, "k_out is q_out"), (dict(k_out=view(2, 2)), INVALID, "k_out is q_in"),
    (dict(q_out=view(4)), INVALID, "q_out is k_in"), (dict(q_gamma=3 * AT + 64), INVALID, "q_out overlaps q_gamma"), (dict(k_gamma=5 * AT), INVALID, "k_out is k_gamma"),
])
def test_head_norm_refusals(host, changed, code, says):
    refused(host, "bl_head_norm_rotary", [table(), norm_args(**changed)], code, says)


@pytest.mark.parametrize("changed,more,code,says", [(c, {}, code, says) for c, code, says in NORM_REFUSALS] + [
    ({}, dict(dq_in=view(8, 2)), INVALID, "overlap"), ({}, dict(dq_in=ops.Heads(6 * AT, 512, 64)), INVALID, "dq_in is dq_out with other strides"),
    ({}, dict(dq_in=ops.Heads(2 * AT, 512, 64)), INVALID, "dq_in is q_in with other strides"), ({}, dict(dq_in=view(7)), INVALID, "dq_in is dk_out"),
    ({}, dict(dk_in=view(8, 2)), INVALID, "dk_in is dq_in"), ({}, dict(dk_in=view(6, 2)), INVALID, "dk_in is dq_out"), ({}, dict(dk_in=view(2, 2)), INVALID, "dk_in is q_in"),
    ({}, dict(workspace_bytes=8), LARGE, "workspace"), ({}, dict(workspace=None), MISALIGNED, "workspace"), ({}, dict(workspace=AT + 8), MISALIGNED, "workspace"),
    ({}, dict(d_q_gamma=AT + 2), MISALIGNED, "d_q_gamma"), ({}, dict(dk_out=ops.Heads(None, 128, 64)), INVALID, "dk_out is null"),
    (dict(q_gamma=8 * AT), {}, INVALID, "dq_in is q_gamma"),
])
def test_head_norm_backward_refusals(host, changed, more, code, says):
    refused(host, "bl_head_norm_rotary_backward", [table(), norm_args(**changed), norm_grads(**more)], code, says)


def test_head_norms_accepted(host):
    both = lambda changed={}, more={}, t=table(): (accepted(host, "bl_head_norm_rotary", [t, norm_args(**changed)]),  # noqa: E731
                                                  accepted(host, "bl_head_norm_rotary_backward", [t, norm_args(**changed), norm_grads(**more)]))
    both()
    both(dict(q_gamma=None, k_gamma=None), dict(d_q_gamma=None, d_k_gamma=None))
    both(dict(positions=None), t=None)  # norms alone
    accepted(host, "bl_head_norm_rotary", [table(), norm_args(q_out=view(2), k_out=view(4, 2))])
    both(more=dict(dq_in=view(6), dk_in=view(4, 2)))
    both(dict(k_heads=0, k_in=ops.Heads(), k_out=ops.Heads(), k_gamma=3), dict(dk_out=ops.Heads(), dk_in=ops.Heads()))
    accepted(host, "bl_head_norm_rotary", [table(), norm_args(rows=0, positions=None)], 0)
    accepted(host, "bl_head_norm_rotary_backward", [table(), norm_args(rows=0, positions=None), norm_grads()], 1)  # the weights' zeros
    n = C.c_uint64()
    assert host.bl_head_norm_rotary_backward_workspace(host.stand_in_ctx(), C.byref(norm_args()), C.byref(n)) == hip.OK and n.value == 9 * 2 * 64 * 4
    assert host.bl_head_norm_rotary_backward_workspace(host.stand_in_ctx(), C.byref(norm_args()), None) == INVALID
    assert host.bl_head_norm_rotary(None, None, C.byref(norm_args())) == INVALID
    assert host.bl_head_norm_rotary(host.stand_in_ctx(), None, None) == INVALID


CACHE_REFUSALS = [
    (dict(cache__kind=2), INVALID, "cache kind"), (dict(head_dim=60), INVALID, "multiple of"), (dict(head_dim=0), INVALID, "multiple of"),
    (dict(head_dim=136), LARGE, "heads of 136"), (dict(cache__page_rows=0), INVALID, "pages of 0"), (dict(cache__page_rows=24), INVALID, "pages of 24"),
    (dict(cache__page_rows=272), LARGE, "pages of 272"), (dict(cache__max_pages=0), INVALID, "no pages"), (dict(cache__max_pages=(1 << 20) + 1), LARGE, "pages of 16"),
    (dict(cache__pages=2**31), LARGE, "in all"), (dict(documents=0), INVALID, "no documents"), (dict(documents=1 << 25), LARGE, "documents"),
    (dict(cache__table=None), INVALID, "table"), (dict(cache__lengths=AT + 2), INVALID, "lengths"), (dict(cache__k__data=None), INVALID, "keys are null"),
    (dict(cache__v__data=21 * AT + 2), MISALIGNED, "values"), (dict(cache__k__row_stride=130), MISALIGNED, "keys"), (dict(cache__v__head_stride=(1 << 41)), LARGE, "values"),
    (dict(cache__k__row_stride=(1 << 25)), LARGE, "keys"), (dict(cache__k__page_stride=1 << 40, cache__pages=1 << 30), LARGE, "keys"),
]


@pytest.mark.parametrize("kind", [ops.CACHE_PLAIN, ops.CACHE_INT4])
@pytest.mark.parametrize("changed,code,says", CACHE_REFUSALS)
def test_cache_refusals(host, kind, changed, code, says):
    refused(host, "bl_cache_append", [table(), append_args(kind, **changed)], code, says)
    refused(host, "bl_cache_read", [read_args(kind, **changed)], code, says)
    refused(host, "bl_paged_attention", [attention_args(kind, **changed)], code, says)


@pytest.mark.parametrize("changed,code,says", [
    (dict(dtype=7), INVALID, "dtype"), (dict(norm=3), INVALID, "norm 3"), (dict(epsilon=math.nan), INVALID, "epsilon"), (dict(kv_heads=0), INVALID, "no key heads"),
    (dict(rows=2**31), LARGE, "rows"), (dict(q_offsets=None), INVALID, "without offsets"), (dict(q_offsets=AT + 2), MISALIGNED, "offsets"),
    (dict(positions=AT + 1), INVALID, "positions"), (dict(q_gamma=AT + 1), MISALIGNED, "q_gamma"), (dict(v_in=ops.Heads(None, 128, 64)), INVALID, "v_in is null"),
    (dict(q_out=ops.Heads(2 * AT, 512, 64)), INVALID, "other strides"), (dict(q_out=view(4)), INVALID, "q_out is k_in"), (dict(q_out=view(5)), INVALID, "q_out is v_in"),
    (dict(q_gamma=3 * AT), INVALID, "q_out is q_gamma"), (dict(cache__k__data=3 * AT), INVALID, "keys is q_out"), (dict(cache__v__data=5 * AT), INVALID, "values is v_in"),
    (dict(cache__k__row_stride=64), INVALID, "overlap"), (dict(cache__v__head_stride=1024), INVALID, "overlap"), (dict(cache__k__page_stride=2048), INVALID, "overlap"),
    (dict(cache__v__data=20 * AT), INVALID, "keys and values overlap"), (dict(cache__v__data=20 * AT + 128), INVALID, "keys and values overlap"),
])
def test_append_refusals(host, changed, code, says):
    refused(host, "bl_cache_append", [table(), append_args(**changed)], code, says)


def test_append_accepted(host):
    for kind in (ops.CACHE_PLAIN, ops.CACHE_INT4):
        accepted(host, "bl_cache_append", [table(), append_args(kind)])
        accepted(host, "bl_cache_append", [None, append_args(kind, norm=0, epsilon=math.nan, q_gamma=1, k_gamma=1)])  # neither is looked at
        accepted(host, "bl_cache_append", [table(), append_args(kind, q_out=view(2))])
        accepted(host, "bl_cache_append", [table(), append_args(kind, q_heads=0, q_in=ops.Heads(), q_out=ops.Heads())])
        accepted(host, "bl_cache_append", [table(), append_args(kind, documents=1, q_offsets=None)])
        accepted(host, "bl_cache_append", [table(), append_args(kind, rows=0)], 0)
        accepted(host, "bl_cache_append", [table(), append_args(kind, cache__pages=0, cache__k__data=None, cache__v__data=None)])
    two = ops.rotary_table([8, 8], 100.0)
    refused(host, "bl_cache_append", [two, append_args()], INVALID, "positions are null")  # a key's index has one axis
    accepted(host, "bl_cache_append", [two, append_args(positions=AT)])
    # Keys and values of a row side by side, and by turns of pages.
    accepted(host, "bl_cache_append", [table(), append_args(cache__k=ops.Pages(20 * AT, 16 * 512, 512, 256), cache__v=ops.Pages(20 * AT + 128, 16 * 512, 512, 256))])
    accepted(host, "bl_cache_append", [table(), append_args(cache__k=ops.Pages(20 * AT, 8192, 128, 2048), cache__v=ops.Pages(20 * AT + 4096, 8192, 128, 2048))])


@pytest.mark.parametrize("changed,code,says", [
    (dict(dtype=7), INVALID, "dtype"), (dict(kv_heads=0), INVALID, "no key heads"), (dict(rows=2**31), LARGE, "rows"), (dict(offsets=None), INVALID, "without offsets"),
    (dict(first=AT + 1), MISALIGNED, "first"), (dict(k_out=ops.Heads(4 * AT + 8, 128, 64)), MISALIGNED, "k_out"), (dict(v_out=ops.Heads(5 * AT, 128, 32)), INVALID, "overlap"),
    (dict(v_out=view(4, 2)), INVALID, "v_out is k_out"), (dict(k_out=view(20, 2)), INVALID, "k_out is the cache's keys"), (dict(k_out=ops.Heads(21 * AT + 64, 128, 64)), INVALID, "overlaps"),
])
def test_read_refusals(host, changed, code, says):
    refused(host, "bl_cache_read", [read_args(**changed)], code, says)


def test_read_accepted(host):
    accepted(host, "bl_cache_read", [read_args()])
    accepted(host, "bl_cache_read", [read_args(first=AT)])
    accepted(host, "bl_cache_read", [read_args(ops.CACHE_INT4, dtype=hip.F32)])
    accepted(host, "bl_cache_read", [read_args(rows=0)], 0)


@pytest.mark.parametrize("changed,code,says", [
    (dict(dtype=7), INVALID, "dtype"), (dict(q_heads=3), INVALID, "3 query heads"), (dict(kv_heads=0), INVALID, "key heads"), (dict(mask=2), INVALID, "mask 2"),
    (dict(mask=0, window=5), INVALID, "window"), (dict(scale=math.nan), INVALID, "scale"), (dict(softcap=-1.0), INVALID, "softcap"), (dict(scale=3e38), INVALID, "beyond f32"),
    (dict(scale=1e30, softcap=1e-30), INVALID, "beyond f32"), (dict(q_rows=1 << 30), LARGE, "query rows"), (dict(q_offsets=None), INVALID, "without offsets"),
    (dict(lse=AT + 2), MISALIGNED, "lse"), (dict(q=ops.Heads(2 * AT + 8, 256, 64)), MISALIGNED, "q's"), (dict(out=ops.Heads(3 * AT, 256, 32)), INVALID, "overlap"),
    (dict(out=view(2)), INVALID, "out is q"), (dict(out=ops.Heads(20 * AT + 128, 256, 64)), INVALID, "out overlaps the cache's keys"), (dict(workspace_bytes=0), LARGE, "workspace"),
    (dict(workspace=None), MISALIGNED, "workspace"), (dict(workspace=AT + 4), MISALIGNED, "workspace"),
])
def test_attention_refusals(host, changed, code, says):
    refused(host, "bl_paged_attention", [attention_args(cache__max_pages=500, **changed)], code, says)


def test_attention_accepted(host):
    for kind in (ops.CACHE_PLAIN, ops.CACHE_INT4):
        for dtype in (hip.F32, hip.F16, ops.BF16):
            wide = {} if kind == ops.CACHE_INT4 or dtype != hip.F32 else dict(cache__k=ops.Pages(20 * AT, 8192, 256, 4096), cache__v=ops.Pages(21 * AT, 8192, 256, 4096))
            accepted(host, "bl_paged_attention", [attention_args(kind, dtype=dtype, **wide)])
        accepted(host, "bl_paged_attention", [attention_args(kind, lse=None, window=3, softcap=5.0)])
        accepted(host, "bl_paged_attention", [attention_args(kind, mask=ops.MASK_NONE, documents=1, q_offsets=None)])
        accepted(host, "bl_paged_attention", [attention_args(kind, q_rows=0)], 0)
    n = C.c_uint64()
    assert host.bl_paged_attention_workspace(host.stand_in_ctx(), C.byref(attention_args(workspace=None, cache__max_pages=500)), C.byref(n)) == hip.OK and n.value > 0
    assert host.bl_paged_attention_workspace(host.stand_in_ctx(), C.byref(attention_args()), None) == INVALID
    assert host.bl_paged_attention(None, C.byref(attention_args())) == INVALID


def test_grids_stay_below_what_a_launch_takes(host):
    """(queries, documents, heads) up to the limits: accepted or refused, never a grid of 2^32 threads."""
    refused(host, "bl_paged_attention", [attention_args(q_rows=1 << 28, q_heads=2, kv_heads=2, out=ops.Heads(3 << 50, 128, 64), q=ops.Heads(2 << 50, 128, 64))], LARGE, "query rows")
    refused(host, "bl_paged_attention", [attention_args(documents=1 << 24, q_heads=64, kv_heads=64)], LARGE, "documents")


# ---- what the calls make of the runtime's answers ----

CACHE_CALLS = r"""
pages = lambda at: ops.Pages(at * AT, 1 << 20, 128, 2048)
def paged(n): return ops.PagedCache(kind=0, pages=100, page_rows=16, max_pages=n, table=AT, lengths=AT, k=pages(20), v=pages(21))
heads = ops.HeadNormArgs(dtype=hip.F16, rows=9, q_heads=4, k_heads=2, head_dim=64, norm=1, epsilon=1e-6, positions=AT, q_in=view(2, 256), q_out=view(3, 256),
                         k_in=view(4, 128), k_out=view(5, 128))
heads_grads = ops.HeadNormGrads(dq_out=view(6, 256), dk_out=view(7, 128), dq_in=view(8, 256), dk_in=view(9, 128), d_q_gamma=AT, workspace=AT, workspace_bytes=1 << 20)
append = ops.CacheAppendArgs(dtype=hip.F16, rows=9, documents=1, q_heads=4, kv_heads=2, head_dim=64, norm=1, epsilon=1e-6, q_in=view(2, 256), q_out=view(3, 256),
                             k_in=view(4, 128), v_in=view(5, 128), cache=paged(4))
read = ops.CacheReadArgs(dtype=hip.F16, rows=9, documents=1, kv_heads=2, head_dim=64, k_out=view(4, 128), v_out=view(5, 128), cache=paged(4))
def paged_attention(n, documents):
    return ops.PagedAttentionArgs(dtype=ops.BF16, q_heads=4, kv_heads=2, head_dim=64, q_rows=documents, documents=documents, scale=0.125, q_offsets=AT, q=view(2, 256), out=view(3, 256),
                                  cache=paged(n), workspace=AT, workspace_bytes=1 << 34)
CALLS.clear()
CALLS.update({
    "heads": (lambda c: ops.head_norm_rotary(c, table, heads), 1),
    "heads backward": (lambda c: ops.head_norm_rotary_backward(c, table, heads, heads_grads), 2),
    "append": (lambda c: ops.cache_append(c, table, append), 1),
    "read": (lambda c: ops.cache_read(c, read), 1),
    "attention": (lambda c: ops.paged_attention(c, paged_attention(1, 2)), 1),
    "attention split": (lambda c: ops.paged_attention(c, paged_attention(4000, 2)), 2),
})
"""


def test_a_host_s_earlier_error_and_device_are_its_own(run):  # noqa: F811
    run(CACHE_CALLS + """
for mine, device in ((0, 0), (0, 1), (1, 0)):
    current.value = mine
    c = hip.Context(device, stream=16 * (device + 1))
    for name, (call, expected) in CALLS.items():
        launches.value, pending.value = 0, 101
        call(c)
        assert (launches.value, pending.value, current.value) == (expected, 101, mine), (name, launches.value, expected)
    pending.value = 0
    c.close()
""")


def test_a_launch_that_fails_is_the_call_s(run):  # noqa: F811
    run(CACHE_CALLS + """
c = hip.Context(0, stream=16)
for name, (call, expected) in CALLS.items():
    for n in range(expected):
        launches.value, failing.value = 0, n
        try:
            call(c)
        except hip.BackendError as e:
            assert e.code == hip.ERR_HIP and launches.value == n + 1, (name, n, e, launches.value)
        else:
            raise AssertionError((name, n))
    failing.value = -1
""")
