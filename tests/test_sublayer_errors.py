"""What the packed sublayer's operators make of the HIP runtime's answers: the
built library, over a stand-in for the runtime's calls that knows two devices
and fails where a test says so. No GPU."""

import pathlib
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent

STAND_IN = r"""
#include <hip/hip_runtime_api.h>
#include <string.h>
extern "C" {
int launches = 0, failing = -1, current = 0;
int calls = 0, elsewhere = 0, at_device = 0;  // calls that ask for a current device, and those of them on another
static hipError_t on_device(void) { calls++; elsewhere += current != at_device; return hipSuccess; }
hipError_t pending = hipSuccess;  // the host thread's last error
static hipError_t failed(hipError_t e) { return pending = e; }
hipError_t hipGetLastError(void) { const hipError_t e = pending; pending = hipSuccess; return e; }
hipError_t hipPeekAtLastError(void) { return pending; }
hipError_t hipGetDeviceCount(int *n) { *n = 2; return hipSuccess; }
hipError_t hipGetDevice(int *d) { *d = current; return hipSuccess; }
hipError_t hipSetDevice(int d) { if (d < 0 || d > 1) return failed(hipErrorInvalidDevice); current = d; return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) {
    memset(p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    p->warpSize = 64;
    p->totalGlobalMem = 1 << 26;
    p->sharedMemPerBlock = 1 << 16;
    p->maxThreadsPerBlock = 1024;
    for (int n = 0; n < 3; n++) p->maxThreadsDim[n] = 1024, p->maxGridSize[n] = 1 << 30;
    return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) { *v = 100000; return hipSuccess; }
// A stream's address is its device's number times 16, and 16; others are no streams.
hipError_t hipStreamGetDevice(hipStream_t s, hipDevice_t *d) {
    if ((size_t)s != 16 && (size_t)s != 32) return failed(hipErrorInvalidHandle);
    *d = (int)((size_t)s / 16) - 1;
    return hipSuccess;
}
// What a program needs beside that: memory, copies and events.
static char memory[1 << 26];
hipError_t hipMalloc(void **p, size_t n) { *p = memory; return n > sizeof memory ? failed(hipErrorOutOfMemory) : on_device(); }
hipError_t hipFree(void *) { return on_device(); }
hipError_t hipMemcpyAsync(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return on_device(); }
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t) { return on_device(); }
hipError_t hipStreamSynchronize(hipStream_t) { return on_device(); }
hipError_t hipEventCreate(hipEvent_t *e) { *e = (hipEvent_t)memory; return on_device(); }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return on_device(); }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float *ms, hipEvent_t, hipEvent_t) { *ms = 1.0f; return hipSuccess; }
hipError_t hipStreamGetCaptureInfo(hipStream_t, hipStreamCaptureStatus *s, unsigned long long *) { *s = hipStreamCaptureStatusNone; return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3 *, dim3 *, size_t *, hipStream_t *) { return hipSuccess; }
hipError_t hipLaunchKernel(const void *, dim3, dim3, void **, size_t, hipStream_t) {
    on_device();
    return launches++ == failing ? failed(hipErrorOutOfMemory) : hipSuccess;
}
}
"""

PROGRAM = r"""
import ctypes as C
import sys
stand_in = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)  # before the library, whose calls it answers
sys.path.insert(0, sys.argv[2])
from beatlm_amd import hip, ops
launches, failing, current, pending = (C.c_int.in_dll(stand_in, n) for n in ("launches", "failing", "current", "pending"))
AT = 1 << 40  # addresses that nothing looks at
view = lambda at, stride: ops.Heads(at * AT, stride, 64)

norm = ops.LayerNormArgs(dtype=hip.F16, rows=4, cols=20, epsilon=1e-6, x_stride=20, y_stride=20, x=AT, gamma=2 * AT, beta=3 * AT, y=4 * AT, mean=5 * AT, rstd=6 * AT)
norm_grads = ops.LayerNormGrads(dy=7 * AT, dy_stride=20, dx=8 * AT, dx_stride=20, d_gamma=9 * AT, d_beta=10 * AT, workspace=11 * AT, workspace_bytes=1 << 30)
turn = ops.RotaryArgs(dtype=hip.F32, rows=9, q_heads=4, k_heads=2, head_dim=64, positions=AT, q_in=view(2, 256), q_out=view(3, 256), k_in=view(4, 128), k_out=view(5, 128))
table = ops.rotary_table([16], 100.0)
def attention(dtype, rows):
    return ops.AttentionArgs(dtype=dtype, q_heads=4, kv_heads=2, head_dim=64, q_rows=rows, k_rows=rows, documents=1, scale=0.125, slopes=AT, q=view(2, 256), k=view(3, 128),
                             v=view(4, 128), out=view(5, 256), lse=6 * AT, workspace=7 * AT, workspace_bytes=1 << 34)
grads = ops.AttentionGrads(d_out=view(8, 256), d_q=view(9, 256), d_k=view(10, 128), d_v=view(11, 128), d_slopes=12 * AT)
CALLS = {  # name: (the call, its launches)
    "norm": (lambda c: ops.layer_norm(c, norm), 1),
    "norm backward": (lambda c: ops.layer_norm_backward(c, norm, norm_grads), 2),
    "rotary": (lambda c: ops.rotary(c, table, turn), 1),
    "attention": (lambda c: ops.attention(c, attention(ops.BF16, 128 * 256)), 1),
    "attention split": (lambda c: ops.attention(c, attention(hip.F32, 300)), 2),
    "backward": (lambda c: ops.attention_backward(c, attention(ops.BF16, 128 * 512), grads), 3),
    "backward split": (lambda c: ops.attention_backward(c, attention(ops.BF16, 300), grads), 5),
    "backward f16": (lambda c: ops.attention_backward(c, attention(hip.F16, 128 * 512), grads), 4),
    "backward f32": (lambda c: ops.attention_backward(c, attention(hip.F32, 300), grads), 5),
}
exec(sys.stdin.read())
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    d = tmp_path_factory.mktemp("errors")
    (d / "stand_in.cpp").write_text(STAND_IN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", str(d / "stand_in.cpp"),
                    "-o", str(d / "libstandin.so"), "-w"], check=True)
    (d / "program.py").write_text(PROGRAM)

    def program(text):
        r = subprocess.run([sys.executable, str(d / "program.py"), str(d / "libstandin.so"), str(ROOT)], input=text, capture_output=True, text=True)
        assert r.returncode == 0, r.stderr

    return program


def test_a_host_s_earlier_error_is_not_the_call_s(run):
    """An error of the host's own, not yet asked for: the calls succeed, launch
    all their kernels and leave it to the host."""
    run("""
c = hip.Context(0, stream=16)
for name, (call, expected) in CALLS.items():
    launches.value, pending.value = 0, 101
    call(c)
    assert (launches.value, pending.value) == (expected, 101), (name, launches.value, expected, pending.value)
""")


def test_a_launch_that_fails_is_the_call_s(run):
    """Whichever of a call's launches fails, the call says so and launches no
    more after it."""
    run("""
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
""")


def test_a_context_over_a_host_s_stream_leaves_the_current_device(run):
    run("""
for mine in (0, 1):
    current.value = mine
    for device in (0, 1):
        c = hip.Context(device, stream=16 * (device + 1))
        assert current.value == mine, (mine, device, "made")
        ops.layer_norm(c, norm)
        assert current.value == mine, (mine, device, "used")
        c.close()
        assert current.value == mine, (mine, device, "closed")
        c = hip.Context(device, stream=0)  # the device's default stream
        c.close()
        assert current.value == mine, (mine, device, "default stream")
""")


def test_a_refused_stream_leaves_no_error_behind(run):
    run("""
for stream in (32, 48):  # another device's, and none
    try:
        hip.Context(0, stream=stream)
    except hip.BackendError as e:
        assert e.code == hip.ERR_INVALID_ARGUMENT
    else:
        raise AssertionError(stream)
    assert (pending.value, current.value) == (0, 0), stream
""")


def test_programs_on_a_host_s_stream_leave_the_current_device(run):
    """Everything that a context over another device's stream does happens on
    that device, the default stream's work too, and leaves the host's current."""
    run("""
import numpy as np
from beatlm_amd import ir
calls, elsewhere, at_device = (C.c_int.in_dll(stand_in, n) for n in ("calls", "elsewhere", "at_device"))
for mine, device, stream in ((0, 0, 16), (0, 1, 32), (1, 0, 0), (0, 1, 0)):
    current.value, at_device.value = mine, device
    launches.value = calls.value = elsewhere.value = 0
    def same(what):
        assert (current.value, elsewhere.value) == (mine, 0), (mine, device, stream, what, current.value, elsewhere.value)
    c = hip.Context(device, stream=stream)
    g = ir.Graph()
    g.tensor(0, ir.INPUT, 33 * 64)
    for t in (1, 2):
        g.tensor(t, ir.WEIGHT, 64)
    g.tensor(3, ir.OUTPUT, 33 * 64)
    g.push(ir.op(ir.OP_LAYER_NORM, [0, 1, 2], [33, 64], 1e-6), 3)
    prep = ir.prepare(c, g)
    same("made")
    prep.write(1, np.ones(64, np.float32))
    same("written")
    prep.run()
    same("run")
    t = hip.Timer(c, 4)
    same("a timer")
    t.begin_frame(1)
    prep.kernels.encode(0, 0, t, 7)
    t.render_begin()
    t.render_end()
    t.resolve()
    same("encoded and timed")
    prep.kernels.time(0, repeats=2)
    same("timed alone")
    c.synchronize()
    prep.read(3)
    same("read")
    t.close()
    prep.close()
    c.close()
    same("closed")
    assert launches.value >= 5 and calls.value > launches.value, (launches.value, calls.value)
""")
