"""The packed sublayer's operators where numbers come near the ends of their
types, against their formulas in 64 bits."""

import pytest
import torch

from beatlm_amd import hip, ops
from tests.opsdata import Packed

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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 72, 128])
@pytest.mark.parametrize("queries", [1, 40])
def test_scores_gradients_beyond_the_type_s_range(gpu, dtype, d, queries):
    """Two keys of equal weight whose values are far apart in every channel,
    under gradients of 1: a score's gradient is 2^17, beyond f16, and d_q, a few
    thousand to 2^15, is not."""
    t = Packed([(queries, 2)] * 2, dtype, 2, 1, d, seed=d)
    t.q.zero_()
    t.q[..., 0] = 2.0**-6
    t.k[:] = torch.rand(4, 1, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) - 0.5
    t.k[..., 0] = 0.0  # scores of 0
    t.v[0::2], t.v[1::2] = 2.0**18 / d, -(2.0**18) / d
    t.d_out.fill_(1.0)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    assert float(t.d_q.float().abs().max()) > 1000.0
    t.check(["out", "lse", "d_q", "d_k", "d_v"], True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_gradients_under_large_values(gpu, dtype, d, mask):
    """Values in the ten thousands over few keys, and over many in documents of
    one batch, beside a document of ordinary ones."""
    t = Packed([(3, 2), (5, 5), (40, 40), (70, 300), (20, 20)], dtype, 4, 2, d, mask=mask)
    t.q *= 0.25
    t.k *= 0.25
    t.v[:-20] *= 8192.0
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v"], True)
