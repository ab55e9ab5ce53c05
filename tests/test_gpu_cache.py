"""The cache of pages (include/beatlm_cache.h): what is appended, read back and
attended over, against the formulas in 64 bits: types, orders of pages, lengths,
pages that end inside a tile or are not there, hidden keys that hold anything,
graphs, streams, and the calls run together."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import (EPSILON, KINDS, NORMS, SENTINEL, Cache, Queries, angles, at, from_codes, heads, ints, normed, tiny, to_codes, turn_tolerance,
                             turned)
from tests.opsdata import DTYPES, F32, assert_within, half_step

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


# ---------------------------------------------------------------------------
# appending
# ---------------------------------------------------------------------------


class Append:
    """New rows of documents behind what their caches hold."""

    def __init__(self, cache, n_new, dtype, q_heads, sections=(), neighbours=False, norm="rms", positions=None, seed=3, gap=0, pad=8):
        self.cache, self.n_new, self.q_heads, self.norm, self.neighbours = cache, n_new, q_heads, norm, neighbours
        self.torch_dtype, self.dtype = DTYPES[dtype]
        d = cache.d
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.offset_list = [gap]
        for n in n_new:
            self.offset_list.append(self.offset_list[-1] + n)
        self.rows = rows = self.offset_list[-1] + gap
        self.offsets = ints(self.offset_list)
        kv = cache.kv_heads
        qkv = torch.randn(rows, q_heads + 2 * kv, d + pad, generator=g, device="cuda").to(self.torch_dtype)
        self.q, self.k, self.v = qkv[:, :q_heads, :d], qkv[:, q_heads:q_heads + kv, :d], qkv[:, q_heads + kv:, :d]
        self.q_out = torch.full((rows, q_heads, d), SENTINEL, device="cuda", dtype=self.torch_dtype)
        self.gamma = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(self.torch_dtype) for _ in range(2)]
        self.table = ops.rotary_table(list(sections), 10000.0, neighbours=neighbours) if sections else None
        self.positions = positions

    def args(self):
        c = self.cache
        return ops.CacheAppendArgs(dtype=self.dtype, rows=self.rows, documents=len(self.n_new), q_heads=self.q_heads, kv_heads=c.kv_heads, head_dim=c.d,
                                   norm=NORMS[self.norm], epsilon=EPSILON, q_offsets=at(self.offsets), positions=at(self.positions), q_gamma=at(self.gamma[0]),
                                   k_gamma=at(self.gamma[1]), q_in=heads(self.q), q_out=heads(self.q_out), k_in=heads(self.k), v_in=heads(self.v), cache=c.struct())

    def places(self):
        got = torch.zeros(self.rows, dtype=torch.int64)
        for doc, n in enumerate(self.n_new):
            got[self.offset_list[doc]:self.offset_list[doc + 1]] = torch.arange(self.cache.lengths[doc] - n, self.cache.lengths[doc])
        return got.cuda()

    def check(self, before):
        """q_out, the new rows of the pools, and everything else as it was."""
        c, u, small = self.cache, half_step(self.torch_dtype), tiny(self.torch_dtype)
        positions = self.positions if self.positions is not None else self.places()[:, None]
        one = torch.ones(self.rows, 0, device="cuda", dtype=torch.float64)
        cos, sin = angles(self.table, positions) if self.table else (one, one)
        want = []
        for x, gamma in ((self.q, self.gamma[0]), (self.k, self.gamma[1])):
            n, n_off, _, _ = normed(x.double(), self.norm)
            z = n * gamma.double() if self.norm != "none" else n
            z_off = n_off * gamma.double().abs() + 2 * F32 * z.abs() if self.norm != "none" else n_off
            y = turned(z, cos, sin, self.neighbours)
            want.append((y, u * y.abs() + turn_tolerance(z, z_off, self.table, self.neighbours) + small))
        inside = slice(self.offset_list[0], self.offset_list[-1])
        assert_within(self.q_out[inside], want[0][0][inside], want[0][1][inside], "q_out")
        assert torch.all(self.q_out[:inside.start] == SENTINEL) and torch.all(self.q_out[inside.stop:] == SENTINEL)
        expected = [b.clone() for b in before]
        for doc, n in enumerate(self.n_new):
            for i in range(n):
                j, row = c.lengths[doc] - n + i, self.offset_list[doc] + i
                if not 0 <= j < c.max_pages * c.page:
                    continue
                page = c.table_list[doc][j // c.page]
                if not 0 <= page < c.pages:
                    continue
                for side in range(2):
                    got = c.pools[side][page, j % c.page, :, :c.row_bytes].contiguous()
                    expected[side][page, j % c.page, :, :c.row_bytes] = got  # looked at here, the rest below
                    if c.kind == "int4":
                        # The codes are those of the 64-bit key rounded to f32: equal bytes. (A 64-bit
                        # computation of another order moves a key's f32 in about 2^-20 of cases, and
                        # then a code in 2^-20 of those.)
                        x = (want[0 + 1][0][row] if side == 0 else self.v[row].double()).float()
                        assert torch.equal(got, to_codes(x)), (side, doc, i)
                    elif side == 0:
                        assert_within(got.view(self.torch_dtype), want[1][0][row], want[1][1][row], "k")
                    else:
                        assert torch.equal(got.view(torch.int16 if self.torch_dtype.itemsize == 2 else torch.int32),
                                           self.v[row].contiguous().view(torch.int16 if self.torch_dtype.itemsize == 2 else torch.int32)), "v"
        for side in range(2):
            assert torch.equal(c.pools[side], expected[side]), "something else was written"


APPENDS = [
    # lengths, new, q_heads, kv_heads, d, page, order, gap, sections, neighbours, norm, kinds
    ([7], [7], 4, 2, 128, 16, "heads", 0, [64], False, "rms", ["plain", "int4"]),
    ([40, 1, 300, 33], [1, 1, 1, 1], 8, 4, 128, 32, "heads", 0, [64], False, "rms", ["plain", "int4"]),
    ([100, 0, 17, 64], [20, 0, 17, 3], 6, 3, 64, 48, "rows", 16, [32], True, "centred", ["plain", "int4"]),
    ([5, 31], [5, 2], 2, 2, 96, 16, "rows", 16, [24], True, "none", ["plain", "int4"]),
    ([3, 50], [3, 50], 0, 1, 32, 256, "heads", 0, [16], False, "rms", ["plain", "int4"]),
    ([70, 9], [33, 9], 5, 5, 40, 16, "heads", 32, [7], False, "centred", ["plain"]),
    ([21], [21], 3, 1, 104, 64, "rows", 0, [], False, "none", ["plain"]),
    ([130, 260], [130, 5], 4, 2, 128, 64, "heads", 16, [1], False, "none", ["plain", "int4"]),
    ([600], [600], 12, 4, 64, 16, "rows", 0, [20], False, "rms", ["plain", "int4"]),
    ([1] * 100, [1] * 100, 2, 1, 64, 16, "heads", 0, [32], False, "rms", ["plain"]),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(gpu, dtype, kind, case):
    lengths, new, q_heads, kv_heads, d, page, order, gap, sections, neighbours, norm, kinds = APPENDS[case]
    if kind not in kinds:
        pytest.skip("codes come in groups of 32 channels")
    cache = Cache(lengths, dtype, kind, kv_heads, d, page, order, gap)
    t = Append(cache, new, dtype, q_heads, sections, neighbours, norm, gap=2, pad=1 if case == 7 else 8)
    before = [p.clone() for p in cache.pools]
    ops.cache_append(gpu, t.table, t.args())
    t.check(before)


@pytest.mark.parametrize("kind", list(KINDS))
def test_append_at_given_positions(gpu, kind):
    cache = Cache([30, 20], "bf16", kind, 2, 64, 16)
    t = Append(cache, [3, 20], "bf16", 4, [16, 16], positions=torch.randint(-9, 2_000_000, (23, 2), device="cuda", dtype=torch.int32))
    before = [p.clone() for p in cache.pools]
    ops.cache_append(gpu, t.table, t.args())
    t.check(before)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("bad", [-1, 10**9, -2**31])
def test_append_drops_what_has_no_place(gpu, kind, bad):
    """More new rows than keys, lengths beyond the table, and pages that are not there."""
    cache = Cache([3, 40, 50], "f16", kind, 2, 64, 16, max_pages=4)
    cache.table_list[1][2] = bad  # keys 32 to 39 of the second document
    cache.table.copy_(torch.tensor(cache.table_list))
    cache.lengths[0], cache.lengths[2] = 3, 4 * 16 + 5
    cache.table_list[2][3] = cache.table_list[2][2] if bad == -1 else cache.table_list[2][3]
    cache.length.copy_(torch.tensor(cache.lengths))
    t = Append(cache, [5, 12, 7], "f16", 2, [32])  # two rows before the first key; 28 .. 39; 62 .. 68 of 64
    cache.table.copy_(torch.tensor(cache.table_list))
    before = [p.clone() for p in cache.pools]
    ops.cache_append(gpu, t.table, t.args())
    t.check(before)


@pytest.mark.parametrize("offsets", [[0, 50, 3, 9], [-7, 2**31 - 1, -2**31, 9], [9, 9, 9, 9], [-1, -1, -1, -1]])
@pytest.mark.parametrize("kind", list(KINDS))
def test_append_and_read_with_wrong_offsets_stay_inside(gpu, kind, offsets):
    """Wrong offsets, lengths and pages: no row outside the pools' pages is
    written (the pools' guards, q_out's and k_out's), whatever goes where."""
    cache = Cache([16, 16, 16], "bf16", kind, 2, 64, 16, gap=16)
    t = Append(cache, [3, 3, 3], "bf16", 2, [32])
    whole = torch.full((t.rows + 8, 2, 64), SENTINEL, device="cuda", dtype=torch.bfloat16)
    out = [torch.full((t.rows + 8, 2, 64), SENTINEL, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    t.offsets.copy_(torch.tensor(offsets))
    cache.length.copy_(torch.tensor([2**31 - 1, -2**31, 17]))
    cache.table.copy_(torch.tensor([[2**31 - 1], [-5], [cache.table_list[2][0]]]))
    a = t.args()
    a.q_out = heads(whole[4:-4])
    ops.cache_append(gpu, t.table, a)
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=ops.BF16, rows=t.rows, documents=3, kv_heads=2, head_dim=64, offsets=at(t.offsets), first=None,
                                          k_out=heads(out[0][4:-4]), v_out=heads(out[1][4:-4]), cache=cache.struct()))
    for x in [whole] + out:
        assert torch.all(x[:4] == SENTINEL) and torch.all(x[-4:] == SENTINEL)
    for pool in cache.pools:  # the pieces between the heads' rows
        assert torch.all(pool[..., cache.row_bytes:] == 0xFF)


def test_codes_at_their_borders(gpu):
    """Ties, groups of one value, zeros, the ends of f16's range, and what f16 cannot hold."""
    d = 64
    cache = Cache([8], "f32", "int4", 1, d, 16)
    t = Append(cache, [8], "f32", 0, norm="none", pad=0)
    step = torch.arange(32, device="cuda", dtype=torch.float32)
    rows = torch.zeros(8, d, device="cuda")
    rows[0, :32] = (step % 16) + 0.5 * (step % 16 < 15)  # ties between codes
    rows[0, 0], rows[0, 15] = 0.0, 15.0
    rows[0, 32:] = 3.25  # one value
    rows[1, :32], rows[1, 32:] = 2.0**-24, -(2.0**-26)
    rows[2, :32] = torch.linspace(-65504, 65504, 32, device="cuda")
    rows[2, 32:] = 65504.0
    rows[3, 5], rows[3, 40] = 65505.0, -70000.0  # beyond f16
    rows[4, 0], rows[4, 33] = math.inf, math.nan
    rows[5] = torch.randn(d, device="cuda") * 1e-6
    rows[6] = torch.randn(d, device="cuda") * 1e4
    rows[7, :32] = 1000.0 + step / 1024
    t.k.copy_(rows[:, None])
    t.v.copy_(-rows[:, None])
    ops.cache_append(gpu, None, t.args())
    for side, x in ((0, rows), (1, -rows)):
        for j in range(8):
            got, want = cache.stored(side, 0, j)[0], to_codes(x[j])
            value, wanted = from_codes(got, d), from_codes(want, d)
            assert torch.equal(value.nan_to_num(-1.0), wanted.nan_to_num(-1.0)), (side, j)
            if j in (3, 4):
                assert bool(value.isnan().all())


@pytest.mark.parametrize("kind", list(KINDS))
def test_a_key_s_bits_do_not_depend_on_its_chunk(gpu, kind):
    """Appended alone, in a chunk and in a batch of others: equal bytes."""
    lengths, stored = [37], []
    for pieces in ([37], [1] * 37, [20, 17]):
        cache = Cache(lengths, "bf16", kind, 2, 128, 16)
        whole = Append(cache, [37], "bf16", 4, [64], "rms")
        first = 0
        for n in pieces:
            a = whole.args()
            a.rows, a.q_offsets = n, None
            for name in ("q_in", "q_out", "k_in", "v_in"):
                h = getattr(a, name)
                setattr(a, name, ops.Heads(h.data + first * h.row_stride * 2, h.row_stride, h.head_stride))
            cache.length.copy_(torch.tensor([first + n]))
            ops.cache_append(gpu, whole.table, a)
            first += n
        stored.append([torch.stack([cache.stored(side, 0, j) for j in range(37)]) for side in range(2)] + [whole.q_out.view(torch.int16)])
    assert all(torch.equal(x, y) for other in stored[1:] for x, y in zip(stored[0], other))


# ---------------------------------------------------------------------------
# reading back
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths,kv_heads,d,page,order,first", [
    ([50, 0, 1, 17], 3, 64, 16, "heads", None), ([300, 129], 2, 128, 48, "rows", [250, 3]), ([70], 1, 32, 256, "heads", [-2]), ([33, 64], 5, 96, 16, "rows", [40, 60]),
])
def test_read(gpu, dtype, kind, lengths, kv_heads, d, page, order, first):
    cache = Cache(lengths, dtype, kind, kv_heads, d, page, order, gap=16)
    if len(lengths) > 1:
        cache.table_list[-1][0] = -1  # a page given back: zeros
        cache.table.copy_(torch.tensor(cache.table_list))
    torch_dtype, code = DTYPES[dtype]
    starts = first or [0] * len(lengths)
    room = [max(0, n - s) + (2 if s >= 0 else 0) for n, s in zip(lengths, starts)]  # and two rows too many
    offset_list = [1]
    for n in room:
        offset_list.append(offset_list[-1] + n)
    rows = offset_list[-1] + 1
    out = [torch.full((rows, kv_heads, d + 8), SENTINEL, device="cuda", dtype=torch_dtype) for _ in range(2)]
    offsets, firsts = ints(offset_list), ints(first) if first else None
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=code, rows=rows, documents=len(lengths), kv_heads=kv_heads, head_dim=d, offsets=at(offsets), first=at(firsts),
                                          k_out=heads(out[0][..., :d]), v_out=heads(out[1][..., :d]), cache=cache.struct()))
    for side in range(2):
        want = torch.full((rows, kv_heads, d + 8), SENTINEL, device="cuda", dtype=torch_dtype)
        for doc, n in enumerate(lengths):
            for i in range(room[doc]):
                j = starts[doc] + i
                if 0 <= j < n:
                    missing = len(lengths) > 1 and doc == len(lengths) - 1 and j < page
                    want[offset_list[doc] + i, :, :d] = 0.0 if missing else cache.rows[side][doc][j].to(torch_dtype)
        assert torch.equal(out[side], want), side


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


ATTENTIONS = [
    # lengths, queries, q_heads, kv_heads, d, page, order, options
    ([1], [1], 1, 1, 64, 16, "heads", dict()),
    ([700], [1], 12, 12, 64, 32, "heads", dict()),
    ([1000, 33, 0, 500], [1, 1, 1, 1], 8, 2, 128, 48, "rows", dict(gap=2)),
    ([300, 16, 31, 129], [5, 5, 5, 5], 12, 2, 64, 16, "heads", dict(cap=9.0)),
    ([260, 40, 7], [40, 7, 7], 4, 2, 128, 64, "rows", dict()),
    ([260, 500], [100, 1], 6, 2, 96, 16, "heads", dict(window=70, gap=3)),
    ([400, 90, 64], [3, 90, 1], 4, 4, 32, 16, "rows", dict(window=1)),
    ([200, 77], [9, 77], 6, 3, 128, 256, "heads", dict(mask="none", cap=4.0)),
    ([4, 2, 20], [9, 5, 20], 2, 1, 64, 16, "heads", dict()),  # more queries than keys: rows that see none
    ([2000], [3], 16, 1, 128, 64, "heads", dict(window=900, cap=20.0)),
    ([130], [130], 20, 4, 64, 16, "rows", dict()),
    ([513, 1024, 31], [1, 2, 3], 24, 3, 128, 32, "heads", dict(mask="none")),
]
PLAIN_ONLY = [
    ([300, 17], [2, 17], 6, 2, 40, 16, "heads", dict(gap=1)), ([90], [1], 3, 3, 8, 32, "rows", dict()), ([150, 65], [30, 65], 4, 1, 104, 48, "rows", dict(window=40)),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind,case", [(k, c) for k in KINDS for c in ATTENTIONS + (PLAIN_ONLY if k == "plain" else [])])
def test_paged_attention(gpu, dtype, kind, case):
    lengths, queries, q_heads, kv_heads, d, page, order, options = case
    cache = Cache(lengths, dtype, kind, kv_heads, d, page, order, gap=16)
    t = Queries(cache, queries, dtype, q_heads, **options)
    ops.paged_attention(gpu, t.args(gpu, max(lengths)))
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lengths,queries,q_heads,kv_heads,d,max_keys", [
    ([5000, 1203], [1, 1], 8, 2, 128, 0), ([4500, 9000], [5, 5], 8, 1, 64, 9000), ([4500, 100], [8, 8], 6, 1, 96, 200), ([3000], [200], 4, 2, 128, 0),
    ([3000, 2500], [150, 1], 4, 4, 64, 700), ([512], [1], 4, 4, 128, 512), ([513], [1], 4, 4, 64, 513),
])
def test_splits_and_long_caches(gpu, dtype, kind, lengths, queries, q_heads, kv_heads, d, max_keys):
    """Keys split over workgroups, each kernel's form, and documents longer than the host said."""
    cache = Cache(lengths, dtype, kind, kv_heads, d, 64)
    t = Queries(cache, queries, dtype, q_heads)
    ops.paged_attention(gpu, t.args(gpu, max_keys))
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("options", [dict(mask="causal", window=30), dict(mask="causal"), dict(mask="none")])
@pytest.mark.parametrize("queries", [1, 6, 50])
def test_pages_that_are_not_there_and_keys_of_anything(gpu, dtype, kind, options, queries):
    """A page given back in the middle, and hidden keys and values that are NaN and infinite."""
    lengths = [100, 131]
    cache = Cache(lengths, dtype, kind, 2, 64, 16, gap=16)
    t = Queries(cache, [queries, 1], dtype, 4, **options)
    cache.table_list[0][1], cache.table_list[1][3] = -1, cache.pages
    cache.table.copy_(torch.tensor(cache.table_list))
    # The last query alone sees the last key; the window ends behind the first.
    last = cache.lengths[0] - 1
    for side in range(2):
        bad = torch.full((2, 64), math.inf if side else math.nan, device="cuda")
        rows = to_codes(bad) if kind == "int4" else bad.to(t.torch_dtype).view(torch.uint8)
        if kind == "int4" and side:  # codes that stand for infinities of either sign: low - inf, step finite
            rows = to_codes(torch.ones(2, 64, device="cuda"))
            rows[:, 34::4], rows[:, 35::4] = 0, 0x7C
        if queries > 1 and options["mask"] == "causal":
            cache.stored(side, 0, last).copy_(rows)
            cache.rows[side][0][last] = from_codes(rows, 64) if kind == "int4" else bad.to(t.torch_dtype).double()
        if options.get("window"):
            j = cache.lengths[1] - 1 - 40  # beyond the second document's window
            cache.stored(side, 1, j).copy_(rows)
            cache.rows[side][1][j] = from_codes(rows, 64) if kind == "int4" else bad.to(t.torch_dtype).double()
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference(missing=[(0, 1), (1, 3)])
    # rows that see a NaN key are NaN; the others are their own
    fine = torch.isfinite(out).all(-1)
    assert bool(fine.any())
    assert_within(t.out[fine], out[fine], out_tol[fine], "out")
    seen = torch.isfinite(lse) | (lse == -math.inf)
    assert_within(t.lse[seen], lse[seen], lse_tol[seen], "lse")
    assert not bool(torch.isfinite(t.out[~fine]).all()) or bool(fine.all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", list(KINDS))
def test_infinite_values_reach_the_rows_that_see_them(gpu, dtype, kind):
    """A last value of infinity: the last query's channels are infinite with its sign, the others' finite."""
    cache = Cache([60], dtype, kind, 1, 64, 16)
    t = Queries(cache, [20], dtype, 2)
    x = torch.ones(1, 64, device="cuda")
    if kind == "int4":
        rows = to_codes(x)
        rows[:, 34], rows[:, 35] = 0, 0x7C  # the first group's low: infinity; its step is zero
        value = from_codes(rows, 64)
    else:
        x[:, :32] = math.inf
        rows, value = x.to(t.torch_dtype).view(torch.uint8), x.to(t.torch_dtype).double()
    cache.stored(1, 0, 59).copy_(rows)
    cache.rows[1][0][59] = value
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, _, _ = t.reference()
    assert_within(t.out[:19], out[:19], out_tol[:19], "out")
    assert bool((t.out[19, :, :32] == math.inf).all()) and bool(torch.isfinite(t.out[19, :, 32:]).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_and_scores_far_apart(gpu, dtype, kind, scale):
    cache = Cache([257, 40], dtype, kind, 2, 128, 32)
    t = Queries(cache, [2, 1], dtype, 8, scale=scale)
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("spread", [1e-30, 1e30])
def test_queries_beyond_f16_s_range_over_codes(gpu, dtype, spread):
    """Taken times a power of two of each row, which the scale undoes."""
    cache = Cache([200], dtype, "int4", 1, 64, 16)
    t = Queries(cache, [3], dtype, 4, spread=spread, scale=0.125 / spread)
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("max_keys", [0, 16, 100000])
def test_what_the_host_knows_of_lengths_decides_no_result(gpu, kind, max_keys):
    cache = Cache([900, 100], "f16", kind, 2, 64, 16)
    t = Queries(cache, [1, 4], "f16", 4, lse=False)
    ops.paged_attention(gpu, t.args(gpu, max_keys))
    out, out_tol, _, _ = t.reference()
    assert_within(t.out, out, out_tol, "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("offsets", [[0, 30, 5, 1000], [-7, 2**31 - 1, -2**31, 12], [12, 12, 3, 0], [2**31 - 1] * 4])
def test_wrong_offsets_and_lengths_stay_inside(gpu, dtype, kind, offsets):
    """The output's and the workspace's guards hold, with NaN around the queries and the pages."""
    cache = Cache([64, 64, 64], dtype, kind, 2, 64, 16, gap=16)
    t = Queries(cache, [4, 4, 4], dtype, 4)
    guard = 8
    t.out = torch.full((12 + 2 * guard, 4, 64), SENTINEL, device="cuda", dtype=t.torch_dtype)
    t.lse = torch.full((2 * guard + 4 * 12,), SENTINEL, device="cuda")
    whole_out, whole_lse = t.out, t.lse
    t.out, t.lse = whole_out[guard:-guard], whole_lse[guard:-guard]
    t.offsets.copy_(torch.tensor(offsets))
    for lengths in ([2**31 - 1, -2**31, 64], [64, 1 << 24, 3]):
        cache.length.copy_(torch.tensor(lengths))
        a = t.args(gpu)
        n = a.workspace_bytes
        space = torch.full((n + 512,), 0xA5, device="cuda", dtype=torch.uint8)
        a.workspace = space.data_ptr() + 256
        ops.paged_attention(gpu, a)
        assert torch.all(whole_out[:guard] == SENTINEL) and torch.all(whole_out[-guard:] == SENTINEL)
        assert torch.all(whole_lse[:guard] == SENTINEL) and torch.all(whole_lse[-guard:] == SENTINEL)
        assert torch.all(space[:256] == 0xA5) and torch.all(space[256 + n:] == 0xA5)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("queries", [1, 40])
def test_what_the_workspace_held_does_not_count(gpu, kind, queries):
    """Counts and maxima of earlier calls, here large numbers, with right offsets and with wrong ones."""
    cache = Cache([900, 70, 300], "bf16", kind, 2, 64, 16)
    t = Queries(cache, [queries, 1, queries], "bf16", 8)
    a = t.args(gpu)
    n = a.workspace_bytes
    assert n > 0
    space = torch.full((n // 4 + 128,), 1e9, device="cuda")
    a.workspace = space.data_ptr() + 256
    ops.paged_attention(gpu, a)
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")
    for offsets in ([0, queries, 0, 2 * queries + 1], [1, 0, 0, 2 * queries]):
        t.offsets.copy_(torch.tensor(offsets))
        space.fill_(1e9)
        ops.paged_attention(gpu, a)
        torch.cuda.synchronize()
        assert torch.all(space[:64] == 1e9) and torch.all(space[64 + n // 4:] == 1e9)


@pytest.mark.parametrize("kind", list(KINDS))
def test_pages_beyond_32_bits(gpu, kind):
    """Pages 3 GiB apart, 9 GiB from the first to the last."""
    cache = Cache([64], "f16", kind, 1, 64, 16)
    far = 3 << 30
    pools = []
    for side in range(2):
        pool = torch.empty(3 * far + (1 << 20), device="cuda", dtype=torch.uint8)
        whole = pool.as_strided((4, 16, 1, cache.row_bytes), (far, cache.row_bytes, cache.row_bytes, 1))
        for n in range(4):
            whole[3 - n] = cache.pools[side][cache.table_list[0][n]]
        pools.append((pool, whole))
    cache.pools, cache.pages = [w for _, w in pools], 4
    cache.table_list = [[3, 2, 1, 0]]
    cache.table.copy_(torch.tensor(cache.table_list))
    t = Queries(cache, [1], "f16", 2)
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, _, _ = t.reference()
    assert_within(t.out, out, out_tol, "out")
    back = [torch.zeros(64, 1, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=hip.F16, rows=64, documents=1, kv_heads=1, head_dim=64, k_out=heads(back[0]), v_out=heads(back[1]), cache=cache.struct()))
    assert all(torch.equal(back[side].double(), cache.rows[side][0]) for side in range(2))
    a = Append(cache, [20], "f16", 2, [32])
    before = [cache.pools[side].clone() for side in range(2)]
    ops.cache_append(gpu, a.table, a.args())
    a.check(before)


@pytest.mark.parametrize("kind", list(KINDS))
def test_attention_repeats_bit_for_bit(gpu, kind):
    cache = Cache([3000, 100], "bf16", kind, 2, 128, 64)
    got = []
    for _ in range(3):
        t = Queries(cache, [1, 30], "bf16", 8)
        ops.paged_attention(gpu, t.args(gpu))
        got.append((t.out.clone(), t.lse.clone()))
    assert all(torch.equal(x, y) for other in got[1:] for x, y in zip(got[0], other))


@pytest.mark.parametrize("kind", list(KINDS))
def test_documents_that_share_pages(gpu, kind):
    """A common prompt's pages in three documents' tables."""
    cache = Cache([90, 90, 90], "bf16", kind, 2, 64, 16)
    for doc in (1, 2):
        for n in range(3):
            cache.table_list[doc][n] = cache.table_list[0][n]
        for side in range(2):
            cache.rows[side][doc][:48] = cache.rows[side][0][:48]
    cache.table.copy_(torch.tensor(cache.table_list))
    t = Queries(cache, [1, 2, 3], "bf16", 4)
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, _, _ = t.reference()
    assert_within(t.out, out, out_tol, "out")


@pytest.mark.parametrize("documents,queries", [(64, 1), (65, 1), (70, 30), (3000, 1)])
def test_many_documents(gpu, documents, queries):
    lengths = [queries + i % 40 for i in range(documents)]
    cache = Cache(lengths, "f16", "plain", 1, 64, 16, fill=True)
    t = Queries(cache, [queries if i % 3 else 1 for i in range(documents)], "f16", 2)
    ops.paged_attention(gpu, t.args(gpu))
    out, out_tol, _, _ = t.reference()
    assert_within(t.out, out, out_tol, "out")


# ---------------------------------------------------------------------------
# the calls together
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", list(KINDS))
def test_a_prompt_then_tokens(gpu, dtype, kind):
    """Chunks of two prompts and then single tokens, each step appended and
    attended over: what attention of all tokens at once over the values that the
    cache holds gives."""
    lengths, d, kv, hq = [45, 23], 64, 2, 4
    cache = Cache(lengths, dtype, kind, kv, d, 16)
    steps = [[30, 17], [10, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1]]
    done, whole = [0, 0], [Append(cache, [n], dtype, hq, [32], seed=7 + doc) for doc, n in enumerate(lengths)]
    outs = [torch.zeros(n, hq, d, device="cuda", dtype=DTYPES[dtype][0]) for n in lengths]
    queries = [torch.zeros(n, hq, d, device="cuda", dtype=DTYPES[dtype][0]) for n in lengths]
    for new in steps:
        new = [min(n, total - so_far) for n, total, so_far in zip(new, lengths, done)]
        cache.lengths = [a + b for a, b in zip(done, new)]
        cache.length.copy_(torch.tensor(cache.lengths))
        t = Append(cache, new, dtype, hq, [32])
        for doc in range(2):
            rows = slice(t.offset_list[doc], t.offset_list[doc + 1])
            for name in ("q", "k", "v"):
                getattr(t, name)[rows] = getattr(whole[doc], name)[done[doc]:done[doc] + new[doc]]
        t.gamma = whole[0].gamma
        ops.cache_append(gpu, t.table, t.args())
        q = Queries(cache, new, dtype, hq)
        q.q = t.q_out
        ops.paged_attention(gpu, q.args(gpu))
        for doc in range(2):
            rows, places = slice(t.offset_list[doc], t.offset_list[doc + 1]), slice(done[doc], done[doc] + new[doc])
            outs[doc][places], queries[doc][places] = q.out[rows], q.q[rows]
        done = list(cache.lengths)
    assert done == lengths
    cache.length.copy_(torch.tensor(lengths))
    back = [torch.zeros(sum(lengths), kv, d, device="cuda") for _ in range(2)]
    offsets = ints([0, 45, 68])
    code = hip.F32 if kind == "int4" or dtype == "f32" else ops.BF16
    back = [b.to(torch.float32 if code == hip.F32 else torch.bfloat16) for b in back]
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=code, rows=68, documents=2, kv_heads=kv, head_dim=d, offsets=at(offsets), k_out=heads(back[0]), v_out=heads(back[1]), cache=cache.struct()))
    for side in range(2):
        cache.rows[side] = [back[side][:45].double(), back[side][45:].double()]
    t = Queries(cache, lengths, dtype, hq)
    t.q.copy_(torch.cat(queries))
    out, out_tol, _, _ = t.reference()
    assert_within(torch.cat(outs), out, out_tol, "out")


@pytest.mark.parametrize("kind", list(KINDS))
def test_a_captured_step_replayed_at_other_lengths(gpu, kind):
    """Append and attention in one graph: lengths, tables and inputs change between replays."""
    stream = torch.cuda.Stream()
    ctx = hip.Context(0, stream=stream.cuda_stream)
    cache = Cache([40, 90, 200], "bf16", kind, 2, 64, 16)
    full = list(cache.lengths)
    a = Append(cache, [1, 1, 1], "bf16", 4, [32])
    t = Queries(cache, [1, 1, 1], "bf16", 4)
    t.q = a.q_out
    args = t.args(ctx)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.cache_append(ctx, a.table, a.args())
        ops.paged_attention(ctx, args)
    for n, lengths in enumerate((full, [1, 17, 33], [39, 64, 129], full)):
        cache.lengths = lengths
        cache.length.copy_(torch.tensor(lengths))
        a.q.copy_(torch.randn(a.q.shape, device="cuda"))
        a.k.copy_(torch.randn(a.k.shape, device="cuda"))
        before = [p.clone() for p in cache.pools]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a.check(before)
        back = []
        for side in range(2):
            docs = []
            for doc in range(3):
                rows = torch.stack([cache.stored(side, doc, j) for j in range(lengths[doc])]).contiguous()
                docs.append(from_codes(rows, 64) if kind == "int4" else rows.view(torch.bfloat16).double())
            back.append(docs)
        kept, cache.rows = cache.rows, back
        out, out_tol, _, _ = t.reference()
        cache.rows = kept
        assert_within(t.out, out, out_tol, f"replay {n}")
    ctx.close()


def test_two_streams_at_once(gpu):
    """Two decoding steps over one cache, a workspace each."""
    cache = Cache([5000], "bf16", "int4", 2, 128, 64)
    want = Queries(cache, [1], "bf16", 8)
    ops.paged_attention(gpu, want.args(gpu))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [hip.Context(0, stream=s.cuda_stream) for s in streams]
    tries = [Queries(cache, [1], "bf16", 8) for _ in range(2)]
    args = [t.args(c) for t, c in zip(tries, contexts)]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, a in zip(contexts, args):
            ops.paged_attention(c, a)
    torch.cuda.synchronize()
    assert all(torch.equal(t.out, want.out) for t in tries)
    for c in contexts:
        c.close()


@pytest.mark.parametrize("kind", list(KINDS))
def test_no_rows_and_no_pages(gpu, kind):
    cache = Cache([20, 5], "f16", kind, 2, 64, 16)
    t = Queries(cache, [2, 1], "f16", 4)
    a = t.args(gpu)
    a.q_rows = 0
    ops.paged_attention(gpu, a)
    assert torch.all(t.out == SENTINEL)
    a = t.args(gpu)
    a.cache.pages, a.cache.k.data, a.cache.v.data = 0, None, None  # every page is missing
    ops.paged_attention(gpu, a)
    assert torch.all(t.out == 0) and torch.all(t.lse == -math.inf)
    b = Append(cache, [2, 1], "f16", 4, [32])
    c = b.args()
    c.cache.pages, c.cache.k.data, c.cache.v.data = 0, None, None
    ops.cache_append(gpu, b.table, c)  # the queries are turned all the same
    assert not bool((b.q_out == SENTINEL).all())


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("queries", [2, 90])
def test_one_document_without_offsets(gpu, kind, queries):
    cache = Cache([700], "bf16", kind, 2, 64, 32)
    t = Queries(cache, [queries], "bf16", 4)
    a = t.args(gpu)
    a.q_offsets = None
    ops.paged_attention(gpu, a)
    out, out_tol, lse, lse_tol = t.reference()
    assert_within(t.out, out, out_tol, "out")
    assert_within(t.lse, lse, lse_tol, "lse")


@pytest.mark.parametrize("kind", list(KINDS))
def test_keys_and_values_side_by_side_among_layers(gpu, kind):
    """One allocation holds two layers' pages, each row's key and value beside each
    other: append, attention and read go by strides, and touch their own layer alone."""
    d, page, kv, pages = 64, 16, 2, 6
    row = 40 if kind == "int4" else 128
    arena = torch.full((pages, 2, page, kv, 2, row), 0xFF, device="cuda", dtype=torch.uint8)
    cache = Cache([50, 20], "f16", kind, kv, d, page, max_pages=4)
    cache.pages, cache.table_list = pages, [[5, 1, 2, 0], [3, 4, -1, -1]]
    cache.table.copy_(torch.tensor(cache.table_list))
    cache.pools = [arena[:, 1, :, :, side] for side in range(2)]
    t = Append(cache, [50, 20], "f16", 4, [32])
    other = arena[:, 0].clone()
    before = [p.clone() for p in cache.pools]
    ops.cache_append(gpu, t.table, t.args())
    t.check(before)
    assert torch.equal(arena[:, 0], other)
    back = [torch.zeros(70, kv, d, device="cuda", dtype=torch.float16) for _ in range(2)]
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=hip.F16, rows=70, documents=2, kv_heads=kv, head_dim=d, offsets=at(t.offsets), k_out=heads(back[0]),
                                          v_out=heads(back[1]), cache=cache.struct()))
    cache.rows = [[b[:50].double(), b[50:].double()] for b in back]
    q = Queries(cache, [3, 20], "f16", 4)
    ops.paged_attention(gpu, q.args(gpu))
    out, out_tol, _, _ = q.reference()
    assert_within(q.out, out, out_tol, "out")
