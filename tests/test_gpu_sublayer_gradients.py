"""Packed attention's gradients against two things that do not know their
formula: autograd through the 64-bit forward, element by element, and
differences of the forward's own outputs."""

import pytest
import torch

from beatlm_amd import hip, ops
from tests.opsdata import Packed, assert_within
from tests.test_sublayer_gradients import CAP, LENS, ROUNDING, SCALE, STEP, difference, direction, heads_of, plain_forward, problem, truncation, value_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    """A context over torch's default stream."""
    try:
        c = hip.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    except (hip.BackendError, RuntimeError) as e:
        pytest.skip(f"no GPU visible: {e}")
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens,q_heads,kv_heads,d,options", [
    ([(40, 40), (21, 21)], 4, 2, 32, dict(mask="causal", cap=1.5, bias=0.2)),
    ([(70, 70), (3, 3)], 6, 2, 64, dict(mask="causal")),
    ([(9, 50), (33, 140)], 2, 1, 128, dict(mask="causal", cap=2.0, spread=2.0)),
    ([(64, 64), (90, 90)], 3, 3, 40, dict(mask="prefix", prefix=[20, 90], bias=0.05)),
    ([(50, 31), (1, 7)], 4, 1, 72, dict(mask="none", cap=1.0, bias=0.1)),
])
def test_gradients_against_autograd(gpu, dtype, lens, q_heads, kv_heads, d, options):
    t = Packed(lens, dtype, q_heads, kv_heads, d, **options)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    leaves = [x.double().requires_grad_() for x in (t.q, t.k, t.v)] + ([] if t.slopes is None else [t.slopes.double().requires_grad_()])
    out = plain_forward(*leaves[:3], lens, t.scale, t.mask, t.cap, *leaves[3:], prefixes=t.prefixes)
    tolerance = t.reference(True)
    for name, want in zip(("d_q", "d_k", "d_v", "d_slopes"), torch.autograd.grad((out * t.d_out.double()).sum(), leaves)):
        value, most = tolerance[name]
        assert_within(value, want, 1e-9 * want.abs().max(), "the tests' own formula: " + name)
        assert_within(getattr(t, name), want, most + 1e-9 * want.abs().max(), name)


@pytest.mark.parametrize("head", range(4))
def test_gradients_along_their_own_signs(gpu, head):
    t = Packed(LENS, "f32", 4, 2, 32, mask="causal", cap=CAP, bias=0.2, scale=SCALE)
    leaves, d_out = problem("cuda")
    for name in leaves:
        getattr(t, name).copy_(leaves[name])
        leaves[name] = getattr(t, name).double()
    t.d_out.zero_()
    t.d_out[:, head] = d_out[:, head]
    d_out = t.d_out.double()
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    off = float((t.reference(False)["out"][1][:, head] * d_out[:, head].abs()).sum())  # of the value

    def value():
        ops.attention(gpu, a)
        return float((t.out[:, head].double() * d_out[:, head]).sum())

    for name in leaves:
        claimed, at = getattr(t, "d_" + name).double(), heads_of(name, head)
        way = direction(claimed, at)
        along = float((claimed * way).sum())
        assert float(claimed.abs().sum()) == along  # nothing for the other heads
        slope = difference(value, getattr(t, name), way.float(), STEP)
        # the two values' errors, and the moved leaf's own rounding, 2^-24 of elements of up to 4, beside a step of 2^-6
        rounding = off / STEP + 2.0**-16 * along
        assert rounding <= ROUNDING[name] * along, (name, rounding, along)
        assert abs(along - slope) <= truncation(value_of(leaves, d_out, head), leaves[name], way) + rounding, (name, along, slope)
