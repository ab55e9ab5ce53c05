"""Caps far beyond the scores: what attention without a cap gives, in every form."""

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import Cache, Queries
from tests.opsdata import DTYPES, F32, assert_within

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


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["plain", "int4"])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e20, 1e38])
@pytest.mark.parametrize("lengths,queries", [([300], [1]), ([2500, 70], [1, 3]), ([400], [12]), ([300, 90], [100, 2])])
def test_wide_caps(gpu, dtype, kind, cap, lengths, queries):
    """cap tanh(s / cap) is s but for s^3 / (3 cap^2), and its steps keep s's own
    digits: a score is off by that and a dozen roundings of itself (of 2^-149 in
    s / cap, for the widest), twice in a probability, once in lse."""
    cache = Cache(lengths, dtype, kind, 2, 64, 16)
    t = Queries(cache, queries, dtype, 4, cap=cap)
    ops.paged_attention(gpu, t.args(gpu, max(lengths)))
    plain = Queries(cache, queries, dtype, 4)
    out, out_tol, lse, lse_tol = plain.reference()
    top = max(float((plain.q.double().norm(dim=-1).max() * k.norm(dim=-1).max()) * plain.scale) for k in cache.rows[0])
    off = top**3 / (3 * cap**2) + 12 * F32 * top + 4 * 2.0**-149 * cap
    worst = max(float(v.abs().max()) for v in cache.rows[1])
    assert_within(t.out, out, out_tol + 2 * off * worst, "out")
    assert_within(t.lse, lse, lse_tol + off, "lse")
