"""Where queries stand whose documents' lengths pass the table's row: the keys
that have no place there are dropped, and every query sees what it would if
they were missing, at the key index it was appended at."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import Cache, Queries, from_codes
from tests.opsdata import assert_within
from tests.test_gpu_cache import Append

pytestmark = pytest.mark.gpu

SLOTS = 64  # 4 pages of 16


@pytest.fixture(scope="module")
def gpu():
    """A context over torch's default stream."""
    try:
        c = hip.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    except (hip.BackendError, RuntimeError) as e:
        pytest.skip(f"no GPU visible: {e}")
    yield c
    c.close()


def appended(gpu, dtype, kind, length, new):
    """A document of `length` keys, `new` of them appended over what 64 slots
    held, beside one that fits; and the queries that were turned with them."""
    cache = Cache([SLOTS, 40], dtype, kind, 2, 64, 16, max_pages=4)
    cache.lengths[0] = length
    cache.length.copy_(torch.tensor(cache.lengths))
    t = Append(cache, [new, 3], dtype, 4, [32])
    before = [p.clone() for p in cache.pools]
    ops.cache_append(gpu, t.table, t.args())
    t.check(before)
    for side in range(2):
        for doc, n in ((0, SLOTS), (1, 40)):
            rows = torch.stack([cache.stored(side, doc, j) for j in range(n)]).contiguous()
            cache.rows[side][doc] = from_codes(rows, 64) if kind == "int4" else rows.view(t.torch_dtype).double()
    return cache, t


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["plain", "int4"])
@pytest.mark.parametrize("window", [0, 10, 30])
@pytest.mark.parametrize("length,new", [(69, 7), (64, 7), (90, 40), (110, 100), (130, 1), (80, 9)])
def test_a_query_stands_where_it_was_appended(gpu, dtype, kind, window, length, new):
    """Few places and many, lengths within and beyond the table, and windows that
    reach into it or lie behind it whole."""
    cache, a = appended(gpu, dtype, kind, length, new)
    beyond = torch.zeros(length - SLOTS, 2, 64, device="cuda", dtype=torch.float64)
    for side in range(2):
        cache.rows[side][0] = torch.cat([cache.rows[side][0], beyond])
    t = Queries(cache, [new, 3], dtype, 4, window=window)
    t.q = a.q_out
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference(missing=[(0, p) for p in range(4, -(-length // 16))])
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("kind", ["plain", "int4"])
@pytest.mark.parametrize("new", [2, 90])
@pytest.mark.parametrize("length", [2**31 - 1, 2**31 - 17, 1 << 24])
def test_lengths_far_beyond_the_table(gpu, kind, new, length):
    """Every key is before every query: all 64 are seen, through a window none."""
    cache = Cache([SLOTS, 40], "bf16", kind, 2, 64, 16, max_pages=4)
    want = Queries(cache, [new, 3], "bf16", 4, mask="none")
    out, out_tol, lse, lse_tol = want.reference()
    cache.length.copy_(torch.tensor([length, 40]))
    rows = slice(0, new)
    t = Queries(cache, [new, 3], "bf16", 4)
    ops.paged_attention(gpu, t.args(gpu))
    assert_within(t.out[rows], out[rows], out_tol[rows], "out")
    assert_within(t.lse[:, rows], lse[:, rows], lse_tol[:, rows], "lse")
    t = Queries(cache, [new, 3], "bf16", 4, window=1000)
    ops.paged_attention(gpu, t.args(gpu))
    assert bool((t.out[rows] == 0).all()) and bool((t.lse[:, rows] == -math.inf).all())
    assert bool(torch.isfinite(t.lse[:, new:]).all())
