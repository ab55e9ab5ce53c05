"""Decoding of bf16 over plain pages is off by its output's own rounding: its
probabilities keep 15 bits."""

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import Cache, Queries
from tests.opsdata import assert_within, half_step

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


@pytest.mark.parametrize("lengths,queries,q_heads,kv_heads,d,options", [
    ([1], [1], 1, 1, 64, dict()), ([300, 41], [1, 1], 8, 2, 128, dict()), ([3000, 700], [1, 1], 12, 12, 64, dict()), ([900], [2], 16, 2, 40, dict()),
    ([5000, 9, 130], [4, 1, 3], 12, 4, 128, dict(window=200)), ([2500], [1], 16, 1, 64, dict(cap=15.0)), ([700], [3], 4, 1, 104, dict(mask="none")),
])
def test_decoding_is_off_by_its_outputs_rounding(gpu, lengths, queries, q_heads, kv_heads, d, options):
    """A probability's first 8 bits are cut off, which leaves under 2^-7 of it, and that
    is rounded to 8 bits: off by 2^-8 2^-7, where the general tolerance allows 2^-8."""
    cache = Cache(lengths, "bf16", "plain", kv_heads, d, 16)
    t = Queries(cache, queries, "bf16", q_heads, **options)
    ops.paged_attention(gpu, t.args(gpu, max(lengths)))
    out, out_tol, lse, lse_tol = t.reference()
    cache.rows[1] = [v.abs() for v in cache.rows[1]]
    whole = t.reference()[0]  # probabilities times the values' magnitudes
    assert_within(t.out, out, out_tol - (half_step(torch.bfloat16) - 2.0**-15) * whole, "out")
    assert_within(t.lse, lse, lse_tol, "lse")
