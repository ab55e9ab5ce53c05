"""Packed attention with offsets that are wrong: nothing outside the tensors
is written or read. Every tensor is an inner slice of a larger one, with
sentinels around what is written and NaN around what is read."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.opsdata import Packed, assert_within

pytestmark = pytest.mark.gpu

ROWS, GUARD, SENTINEL = 64, 40, 7.0


@pytest.fixture(scope="module")
def gpu():
    """A context over torch's default stream."""
    try:
        c = hip.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    except (hip.BackendError, RuntimeError) as e:
        pytest.skip(f"no GPU visible: {e}")
    yield c
    c.close()


class Guarded(Packed):
    """A problem whose tensors have guards: rows before and behind, and values
    before and behind the flat arrays and the workspace."""

    def __init__(self, *args, **options):
        super().__init__(*args, **options)
        self.held = {}
        for name in ("q", "k", "v", "d_out"):
            self.put(name, getattr(self, name), math.nan)
        for name in ("out", "d_q", "d_k", "d_v", "lse", "d_slopes"):
            if getattr(self, name) is not None:
                self.put(name, getattr(self, name), SENTINEL)
        for name in ("q_positions", "k_positions"):
            if getattr(self, name) is not None:
                self.put(name, getattr(self, name), 2**27)

    def put(self, name, tensor, fill):
        # [GUARD | rows of the tensor, as they lie | GUARD] by elements of its first axis; lse and slopes flat
        flat = name in ("lse", "d_slopes")
        kept = tensor.flatten() if flat else tensor
        whole = torch.full((kept.shape[0] + 2 * GUARD, *kept.shape[1:]), fill, device="cuda", dtype=kept.dtype)
        whole[GUARD:GUARD + kept.shape[0]] = kept
        self.held[name] = whole
        setattr(self, name, whole[GUARD:GUARD + kept.shape[0]].view(tensor.shape))

    def ready(self, gpu):
        a = self.args(gpu, True)
        n = a.workspace_bytes
        self.workspace = torch.full((n + 512,), 0xA5, device="cuda", dtype=torch.uint8)
        a.workspace = self.workspace.data_ptr() + 256
        return a

    def check_guards(self):
        for name in ("out", "d_q", "d_k", "d_v", "lse", "d_slopes"):
            if name in self.held:
                whole = self.held[name].float()
                assert torch.all(whole[:GUARD] == SENTINEL) and torch.all(whole[-GUARD:] == SENTINEL), name
        assert torch.all(self.workspace[:256] == 0xA5) and torch.all(self.workspace[-256:] == 0xA5)


OPTIONS = [dict(mask="prefix", bias=0.1), dict(mask="causal", cap=9.0), dict(mask="none", bias=0.1, axes=2), dict(mask="causal")]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("off", [[0, 50, 20, 1000], [-7, 2**31 - 1, -2**31, 64], [60, 60, 10, 0], [2**31 - 1] * 4, [-1, -1, -1, -1], [64, 0, 64, 0]])
def test_wrong_offsets_write_nothing_outside(gpu, dtype, options, d, off):
    t = Guarded([(20, 20), (20, 20), (24, 24)], dtype, 4, 2, d, **options)
    assert (t.q_rows, t.k_rows) == (ROWS, ROWS)
    for q_off, k_off in ((off, off[::-1]), (off, off), (off[::-1], [0, 20, 40, 64])):
        t.q_off.copy_(torch.tensor(q_off))
        t.k_off.copy_(torch.tensor(k_off))
        if t.prefix is not None:
            t.prefix.copy_(torch.tensor([2**31 - 1, -2**31, 5]))
        a = t.ready(gpu)
        ops.attention(gpu, a)
        ops.attention_backward(gpu, a, t.grads())
        t.check_guards()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("d", [64, 128])
def test_offsets_beyond_the_tensors_end_with_them(gpu, dtype, options, d):
    """Rising offsets before the first row and behind the last: the results of
    the clamped ones, with nothing of the NaN around the tensors in them."""
    t = Guarded([(20, 44), (44, 20)], dtype, 4, 2, d, prefix=[11, 3], **options)
    t.q_off.copy_(torch.tensor([-7, 20, 2**31 - 1]))
    t.k_off.copy_(torch.tensor([-2**31, 44, 65]))
    a = t.ready(gpu)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    want = t.reference(True)
    for name in ("out", "lse", "d_q", "d_k", "d_v", "d_slopes"):
        if getattr(t, name) is not None:
            assert_within(getattr(t, name), *want[name], name)
    t.check_guards()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_single_tokens_stay_inside_too(gpu, dtype):
    """The forward over few rows, split keys and a cache with wrong ends."""
    t = Guarded([(1, 700), (1, 300)], dtype, 8, 2, 64, mask="causal", bias=0.1, axes=1)
    for k_off in ([0, 5000, 1000], [-900, 300, 2**31 - 1], [1000, 0, 400]):
        t.k_off.copy_(torch.tensor(k_off))
        a = t.ready(gpu)
        ops.attention(gpu, a)
        t.check_guards()
    t.k_off.copy_(torch.tensor([-3, 700, 1003]))
    ops.attention(gpu, t.ready(gpu))
    want = t.reference(False)
    for name in ("out", "lse"):
        assert_within(getattr(t, name), *want[name], name)
    t.check_guards()
