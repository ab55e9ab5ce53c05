"""What the host side of the heads' norms (csrc/cache_ops.cpp) hands to the
kernels of tensors that have no heads: nothing that a kernel could read."""

import ctypes as C
import subprocess

import pytest

from beatlm_amd import hip, ops
from tests.test_sublayer_cache import AT, MORE, ROOT, norm_args, norm_grads, table
from tests.test_sublayer_ops import STAND_INS

RECORDING = r"""
static const void *handed[2];
extern "C" const void *handed_gamma(int n) { return handed[n]; }
static void keep(const bl::HeadsParams &p) { handed[0] = p.q_gamma, handed[1] = p.k_gamma; }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("weights")
    more = MORE
    for name in ("launch_heads_forward", "launch_heads_backward"):
        plain = f"hipError_t {name}(const HeadsParams &, uint32_t, uint32_t, hipStream_t) {{ return"
        assert plain in more
        more = more.replace(plain, f"hipError_t {name}(const HeadsParams &p, uint32_t, uint32_t, hipStream_t) {{ keep(p); return")
    (d / "stand_ins.cpp").write_text(STAND_INS + RECORDING + more)
    csrc = ROOT / "beatlm_amd" / "csrc"
    subprocess.run(["/opt/rocm/llvm/bin/clang++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", f"-I{csrc}",
                    str(csrc / "cache_ops.cpp"), str(csrc / "paged_plan.cpp"), str(d / "stand_ins.cpp"), "-o", str(d / "libweights.so"), "-Wl,-Bsymbolic", "-w"],
                   check=True)
    lib = C.CDLL(str(d / "libweights.so"))
    lib.stand_in_ctx.restype = lib.handed_gamma.restype = C.c_void_p
    for name, (res, args) in ops._CACHE_SIG.items():
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    return lib


@pytest.mark.parametrize("q_heads,k_heads", [(4, 0), (0, 2), (4, 2)])
def test_weights_of_no_heads_reach_no_kernel(host, q_heads, k_heads):
    """The backward lays both tensors' weights into LDS, whoever has heads: an address
    that the header says is not touched, here one beyond any memory, would be read."""
    nowhere = (1 << 62) + 1
    a = norm_args(q_heads=q_heads, k_heads=k_heads, q_gamma=AT if q_heads else nowhere, k_gamma=AT if k_heads else nowhere)
    want = (AT if q_heads else None, AT if k_heads else None)
    for name, more in (("bl_head_norm_rotary", []), ("bl_head_norm_rotary_backward", [norm_grads()])):
        assert getattr(host, name)(host.stand_in_ctx(), *[C.byref(s) for s in (table(), a, *more)]) == hip.OK
        assert (host.handed_gamma(0), host.handed_gamma(1)) == want, name
