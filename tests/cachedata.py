"""Inputs and 64-bit references for the norms of heads and the cache of pages
(include/beatlm_cache.h): plain torch from the header's formulas, with the
magnitudes that the tolerances are made of (those of tests/opsdata.py)."""

import math

import torch

from beatlm_amd import hip, ops
from tests.opsdata import DTYPES, F32, half_step

NORMS = {"none": ops.HEAD_NORM_NONE, "rms": ops.HEAD_NORM_RMS, "centred": ops.HEAD_NORM_CENTRED}
KINDS = {"plain": ops.CACHE_PLAIN, "int4": ops.CACHE_INT4}
EPSILON = 1e-5
SENTINEL = 7.0


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def at(t):
    return None if t is None else t.data_ptr()


def heads(t):
    return ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))


# ---------------------------------------------------------------------------
# a head's norm and rotation, with what f32 may be off
# ---------------------------------------------------------------------------


def turned(x, cos, sin, neighbours):
    """x [rows][heads][d] by the angles [rows][pairs]; channels beyond the pairs as they are."""
    p = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    y = x.clone()
    first, second = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if neighbours else (slice(0, p), slice(p, 2 * p))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    return y


def spread(size, pairs, neighbours):
    """Of magnitudes: what a rotation mixes, the sum over a pair's two channels."""
    one = torch.ones(size.shape[0], pairs, device=size.device, dtype=torch.float64)
    y = size.clone()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., first] = y[..., second] = (size[..., first] + size[..., second]) * one[:, None]
    return y


def angles(table, positions):
    """cos and sin [rows][pairs] of a rotary table at [rows][axes]."""
    turns = torch.tensor(table.turns[:table.pairs], device=positions.device, dtype=torch.float64)
    axis = torch.tensor(list(table.axis[:table.pairs]), device=positions.device, dtype=torch.long)
    phi = positions.double()[:, axis] * turns * (2 * math.pi)
    return phi.cos(), phi.sin()


def normed(x, norm):
    """(n, its f32 error, rstd, its f32 error) of x in 64 bits. A head's sum is at
    most 16 channels a thread and 6 additions over them: 24 steps, twice as
    many for squares of a mean that is off itself."""
    if norm == "none":
        return x, torch.zeros_like(x), torch.ones_like(x[..., :1]), torch.zeros_like(x[..., :1])
    sums = 48 * F32
    mean = x.mean(-1, keepdim=True) if norm == "centred" else torch.zeros_like(x[..., :1])
    mean_off = sums * x.abs().mean(-1, keepdim=True) if norm == "centred" else torch.zeros_like(mean)
    rstd = (((x - mean) ** 2).mean(-1, keepdim=True) + EPSILON).rsqrt()
    rstd_off = rstd * (sums + 8 * F32 + 2 * mean_off * rstd)
    n = (x - mean) * rstd
    return n, mean_off * rstd + n.abs() * (rstd_off / rstd + 2 * F32) + F32 * x.abs() * rstd, rstd, rstd_off


def turn_tolerance(z, z_off, table, neighbours):
    """Of z turned: its own error mixed, and products and sines good to a few steps."""
    if table is None:
        return z_off
    return spread(z_off + 8 * F32 * z.abs(), table.pairs, neighbours)


def tiny(dtype):
    return 2.0**-25 if dtype == torch.float16 else 1e-37


# ---------------------------------------------------------------------------
# 4-bit codes
# ---------------------------------------------------------------------------


def nibble_places(d):
    """(32-bit word, bits) of each channel's code."""
    c = torch.arange(d)
    return c // 8, c % 8 // 2 * 4 + c % 2 * 16


def to_codes(x):
    """[..., d] in f32 -> rows of bytes, as the header says."""
    d = x.shape[-1]
    g = x.float().unflatten(-1, (-1, 32)).double()
    low, top = g.amin(-1), g.amax(-1)
    bad = ~(g.abs() <= 65504).all(-1)
    step = ((top - low) / 15).float().half().masked_fill(bad, math.nan)
    low = low.float().half()
    code = torch.round((g - low.double()[..., None]) / step.double()[..., None]).nan_to_num(0.0, 15.0, 0.0).clamp(0, 15).long()
    code = code.masked_fill(~(step > 0)[..., None], 0).flatten(-2)
    word, bits = nibble_places(d)
    words = torch.zeros(*x.shape[:-1], d // 8, device=x.device, dtype=torch.long)
    for c in range(d):
        words[..., int(word[c])] |= code[..., c] << int(bits[c])
    words = torch.where(words >= 2**31, words - 2**32, words).to(torch.int32)
    params = torch.stack([step, low], -1).flatten(-2)
    return torch.cat([words.view(torch.uint8), params.view(torch.uint8)], -1)


def from_codes(rows, d):
    """What rows of bytes stand for, in 64 bits."""
    words = rows[..., :d // 2].contiguous().view(torch.int32).long()
    params = rows[..., d // 2:].contiguous().view(torch.float16).double()
    word, bits = nibble_places(d)
    code = torch.stack([words[..., int(word[c])] >> int(bits[c]) & 15 for c in range(d)], -1).double()
    step, low = params[..., 0::2].repeat_interleave(32, -1), params[..., 1::2].repeat_interleave(32, -1)
    return (low + code * step).half().double()


# ---------------------------------------------------------------------------
# a cache of pages
# ---------------------------------------------------------------------------


class Cache:
    """Documents' keys and values [n][heads][d] in pages dealt out at random:
    garbage (NaN, or codes that stand for it) in every row no document has, and
    around the rows, as `gap` bytes between heads."""

    def __init__(self, lengths, dtype, kind, kv_heads, d, page, order="heads", gap=0, seed=1, max_pages=None, fill=True, spread=1.0):
        self.torch_dtype, self.dtype = DTYPES[dtype]
        self.kind, self.kv_heads, self.d, self.page, self.lengths = kind, kv_heads, d, page, list(lengths)
        g = torch.Generator(device="cuda").manual_seed(seed)
        of = [-(-n // page) for n in lengths]
        self.pages = sum(of) + 3
        self.max_pages = max_pages or max(1, max(of))
        self.row_bytes = d // 2 + d // 8 if kind == "int4" else d * self.torch_dtype.itemsize
        piece = self.row_bytes + gap
        shape = (self.pages, kv_heads, page, piece) if order == "heads" else (self.pages, page, kv_heads, piece)
        deal = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table_list = []
        for n in of:
            self.table_list.append([deal.pop() for _ in range(n)] + [-1] * (self.max_pages - n))
        self.table, self.length = ints(self.table_list), ints(self.lengths)
        self.pools, self.rows = [], []  # bytes as [page][row][head][piece]; what they hold
        for _ in range(2):
            pool = torch.full(shape, 0xFF, device="cuda", dtype=torch.uint8)  # NaN in every type
            view = pool if order == "rows" else pool.transpose(1, 2)
            docs = []
            for doc, n in enumerate(lengths):
                x = torch.randn(n, kv_heads, d, generator=g, device="cuda") * spread
                rows = to_codes(x) if kind == "int4" else x.to(self.torch_dtype).contiguous().view(torch.uint8)
                if fill:
                    for j in range(0, n, page):
                        view[self.table_list[doc][j // page], :min(page, n - j), :, :self.row_bytes] = rows[j:j + page]
                docs.append(from_codes(rows, d) if kind == "int4" else x.to(self.torch_dtype).double())
            self.pools.append(view)
            self.rows.append(docs)

    def struct(self):
        side = lambda p: ops.Pages(p.data_ptr(), p.stride(0), p.stride(1), p.stride(2))  # noqa: E731
        return ops.PagedCache(kind=KINDS[self.kind], pages=self.pages, page_rows=self.page, max_pages=self.max_pages, table=at(self.table),
                              lengths=at(self.length), k=side(self.pools[0]), v=side(self.pools[1]))

    def stored(self, side, doc, j):
        """The bytes of a document's key, [head][row_bytes]."""
        return self.pools[side][self.table_list[doc][j // self.page], j % self.page, :, :self.row_bytes]


class Queries:
    """Attention of packed queries over a Cache: spare rows around, NaN in them."""

    def __init__(self, cache, n_q, dtype, q_heads, mask="causal", window=0, cap=0.0, scale=None, seed=2, gap=0, spread=1.0, lse=True):
        self.cache, self.n_q, self.q_heads = cache, n_q, q_heads
        self.torch_dtype, self.dtype = DTYPES[dtype]
        self.mask, self.window, self.cap = mask, window, cap
        d = cache.d
        self.scale = d**-0.5 if scale is None else scale
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.offset_list = [gap]
        for n in n_q:
            self.offset_list.append(self.offset_list[-1] + n)
        rows = self.offset_list[-1] + gap
        self.offsets = ints(self.offset_list)
        self.q = torch.full((rows, q_heads, d), math.nan, device="cuda", dtype=self.torch_dtype)
        self.q[gap:rows - gap] = (torch.randn(rows - 2 * gap, q_heads, d, generator=g, device="cuda") * spread).to(self.torch_dtype)
        self.out = torch.full((rows, q_heads, d), SENTINEL, device="cuda", dtype=self.torch_dtype)
        self.lse = torch.full((q_heads, rows), SENTINEL, device="cuda") if lse else None

    def args(self, ctx, max_keys=0):
        a = ops.PagedAttentionArgs(
            dtype=self.dtype, q_heads=self.q_heads, kv_heads=self.cache.kv_heads, head_dim=self.cache.d, q_rows=self.q.shape[0], documents=len(self.n_q),
            mask=ops.MASK_CAUSAL if self.mask == "causal" else ops.MASK_NONE, window=self.window, max_keys=max_keys, scale=self.scale, softcap=self.cap,
            q_offsets=at(self.offsets), q=heads(self.q), out=heads(self.out), lse=at(self.lse), cache=self.cache.struct())
        n = ops.paged_attention_workspace(ctx, a)
        self.workspace = torch.full((n + 16,), 0xFF, device="cuda", dtype=torch.uint8)  # what it holds means nothing
        a.workspace, a.workspace_bytes = self.workspace.data_ptr(), n
        return a

    def reference(self, missing=()):
        """(out, tolerance, lse, tolerance) in 64 bits; `missing`: (document, page) pairs that are not there.

        A score is off by its product's sum in f32, the cap (a tanh good to a few
        steps of 1, times the cap) and the exponent's argument in base two; f32
        queries over codes are two f16 pieces, 2^-22 of each. Probabilities are
        rounded to the matrix cores' type: u of it, 2^-22 as two pieces."""
        c = self.cache
        u = half_step(self.torch_dtype)
        f32 = self.torch_dtype == torch.float32
        inner = (2.0**-22 if f32 else half_step(torch.float16)) if c.kind == "int4" else (0.0 if f32 else u)
        pieces = 2.0**-22 if f32 and c.kind == "int4" else 2.0**-24
        low = c.kind == "int4" or self.torch_dtype == torch.float16  # probabilities in f16: its subnormals
        out = torch.full(self.out.shape, SENTINEL, device="cuda", dtype=torch.float64)
        lse = torch.full((self.q_heads, self.q.shape[0]), SENTINEL, device="cuda", dtype=torch.float64)
        out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
        group = self.q_heads // c.kv_heads
        for doc, n in enumerate(self.n_q):
            n_k = c.lengths[doc]
            rows = slice(self.offset_list[doc], self.offset_list[doc + 1])
            place = torch.arange(n_k - n, n_k, device="cuda")[:, None]
            j = torch.arange(n_k, device="cuda")[None]
            seen = torch.ones(n, n_k, device="cuda", dtype=torch.bool)
            if self.mask == "causal":
                seen = j <= place
                if self.window:
                    seen = seen & (j > place - self.window)
            for d, p in missing:
                if d == doc:
                    seen = seen & ~((j >= p * c.page) & (j < (p + 1) * c.page))
            for h in range(self.q_heads):
                q, k, v = self.q[rows, h].double(), c.rows[0][doc][:, h // group], c.rows[1][doc][:, h // group]
                raw, size = q @ k.T * self.scale, q.abs() @ k.abs().T * abs(self.scale)
                s = self.cap * torch.tanh(raw / self.cap) if self.cap else raw
                s = s.masked_fill(~seen, -math.inf)
                off = F32 * ((c.d + 4) * size + 8 * self.cap + 4 * s.masked_fill(~seen, 0.0).abs() + 8) + pieces * size
                off = off.masked_fill(~seen, 0.0)
                worst = off.amax(1) if n_k else torch.zeros(n, device="cuda", dtype=torch.float64)
                stat = torch.logsumexp(s, 1) if n_k else torch.full((n,), -math.inf, device="cuda", dtype=torch.float64)
                dead = stat == -math.inf
                p = torch.where(seen, (s - stat.masked_fill(dead, 0.0)[:, None]).exp(), torch.zeros_like(s))
                relative = 2 * (off + worst[:, None] + F32 * (n_k + 16))
                o = torch.where(seen[:, :, None], v[None], torch.zeros_like(v)[None])  # hidden values may be anything
                out[rows, h] = (p[:, None] @ o)[:, 0] if n_k else 0.0
                tol = u * out[rows, h].abs() + 1e-30
                if n_k:
                    tol = tol + ((p * (relative + inner))[:, None] @ o.abs())[:, 0]
                    if low:
                        tol = tol + 2.0**-25 * (2.0**-8 * (seen.double()[:, None] @ o.abs())[:, 0])
                out_tol[rows, h] = tol + (2.0**-25 if self.torch_dtype == torch.float16 else 0.0)
                lse[h, rows] = stat
                lse_tol[h, rows] = worst + F32 * (n_k + 16 + 4 * stat.masked_fill(dead, 0.0).abs())
        return out, out_tol, lse, lse_tol
