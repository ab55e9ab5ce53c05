"""NaN and infinities in keys and values that queries do see, row by row and
channel by channel."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import Cache, Queries, from_codes, to_codes
from tests.opsdata import DTYPES, assert_within

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


FORMS = [([70], [1]), ([70], [9]), ([100], [60]), ([300, 90], [100, 2]), ([1500], [3])]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["plain", "int4"])
@pytest.mark.parametrize("cap", [0.0, 7.0])
@pytest.mark.parametrize("mask", ["causal", "none"])
@pytest.mark.parametrize("lengths,queries", FORMS)
def test_a_nan_key_makes_nan_of_the_rows_that_see_it(gpu, dtype, kind, cap, mask, lengths, queries):
    """All their channels and their lse, of the key's heads alone; the others are their own."""
    cache = Cache(lengths, dtype, kind, 2, 64, 16)
    t = Queries(cache, queries, dtype, 4, mask=mask, cap=cap)
    j = lengths[0] - (queries[0] + 1) // 2  # the later half of a causal document's queries see it
    x = cache.rows[0][0][j].float()
    x[1] = math.nan
    rows = to_codes(x) if kind == "int4" else x.to(t.torch_dtype).contiguous().view(torch.uint8)
    cache.stored(0, 0, j)[1] = rows[1]
    cache.rows[0][0][j, 1] = math.nan
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference()
    nan = out.isnan().any(-1)
    assert bool(nan.any()) and bool((~nan).any()) and not bool(nan[:, :2].any())
    assert bool((nan == lse.T.isnan()).all())
    assert bool(t.out[nan].isnan().all()) and bool(t.lse.T[nan].isnan().all())
    assert_within(t.out[~nan], out[~nan], out_tol[~nan], "out")
    assert_within(t.lse.T[~nan], lse.T[~nan], lse_tol.T[~nan], "lse")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["plain", "int4"])
@pytest.mark.parametrize("cap", [0.0, 7.0])
@pytest.mark.parametrize("mask", ["causal", "none"])
@pytest.mark.parametrize("lengths,queries", FORMS)
def test_infinite_and_nan_values_reach_their_channels(gpu, dtype, kind, cap, mask, lengths, queries):
    """Infinities of both signs and NaN, apart and against each other, in the rows that see them."""
    cache = Cache(lengths, dtype, kind, 2, 64, 16)
    t = Queries(cache, queries, dtype, 4, mask=mask, cap=cap)
    last = lengths[0] - 1
    puts = [(last, 1, 0, math.inf), (last - 20, 1, 1, -math.inf), (last - 1, 0, 0, math.nan), (last - 21, 0, 1, -math.inf), (last - 18, 0, 1, math.inf)]
    for j, head, group, value in puts:
        if kind == "int4":  # a group of 32 channels: its low, with a step of zero
            low = torch.tensor([0.0, value], device="cuda", dtype=torch.float16).view(torch.uint8)
            cache.stored(1, 0, j)[head, 32 + 4 * group:36 + 4 * group] = low
            cache.rows[1][0][j, head] = from_codes(cache.stored(1, 0, j)[head], 64)
        else:
            x = cache.stored(1, 0, j)[head].clone().view(t.torch_dtype)
            x[32 * group:32 * group + 5] = value
            cache.stored(1, 0, j)[head] = x.view(torch.uint8)
            cache.rows[1][0][j, head] = x.double()
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference()
    fine = torch.isfinite(out)
    assert not bool(fine.all())
    assert bool((t.out.isnan() == out.isnan()).all())
    assert bool(((t.out == math.inf) == (out == math.inf)).all()) and bool(((t.out == -math.inf) == (out == -math.inf)).all())
    assert_within(t.out[fine], out[fine], out_tol[fine], "out")
    assert_within(t.lse, lse, lse_tol, "lse")
