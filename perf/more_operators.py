"""What the operators of a paged key cache are measured on (beatlm_amd.ops):
norms of queries and keys for each head with their rotary positions in the same
pass, and the gradients; new keys and values normed, turned and appended to
pages that hold the tensors' type or 4-bit codes; and attention over such pages,
from one decoded token to chunks of prompts.

A case is a dict of plain values:

  op       "heads", "append" or "attention"
  dtype    "f32", "f16" or "bf16"

  heads:     `rows` tokens, `q_heads` + `k_heads` heads of `head_dim`, of which
             `pairs` pairs turn; `norm` "rms" or "centred"; `axes` (1 text, 2
             images, 3 video); `layout` "halves" or "neighbours"; `start` the
             first position; `train`: the forward and the backward
  append:    `documents` documents of up to `queries` new tokens each behind up
             to `past` cached ones (`ragged` 0: all the longest), `kind` "plain"
             or "int4" pages of `page` tokens, `order` "heads" ([page][head][token])
             or "rows" ([page][token][head]); `norm` "none", "rms" or "centred"
  attention: `documents` documents of `queries` query tokens each (`mixed` 1: every
             second has one) over up to `keys` cached ones; `mask` "none" or
             "causal"; `window` the nearest keys a query sees (0: all); `cap`
             the bound of the scores (0: none); `spare` rows behind the last
             document

A row of 4-bit codes, for a token and a key head: head_dim / 2 bytes, channel 2 n
of each 8 in bits 4 n of 32, channel 2 n + 1 in bits 16 + 4 n, then a step and a
low (f16) for each 32 channels. A code stands for f16(low + code * step).
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPSILON = 1e-6
BASE = 10000.0
GROUP = 32
NIBBLES = [0, 4, 1, 5, 2, 6, 3, 7]  # of 32 bits, in the channels' order
_context = None


def listed():
    return [
        # Eight sequences' next tokens between two kernels of a decoding step: latency alone.
        {"name": "heads_tokens_f16", "op": "heads", "dtype": "f16", "train": False, "rows": 8, "q_heads": 16, "k_heads": 4, "head_dim": 128,
         "pairs": 64, "norm": "rms", "axes": 1, "layout": "halves", "start": 5000},
        # A training step's queries and keys of a long text, key heads shared.
        {"name": "heads_train_bf16", "op": "heads", "dtype": "bf16", "train": True, "rows": 32768, "q_heads": 16, "k_heads": 4, "head_dim": 128,
         "pairs": 64, "norm": "rms", "axes": 1, "layout": "halves", "start": 0},
        # Images' rows and columns in full precision, an odd head of which a part turns.
        {"name": "heads_train_odd_f32", "op": "heads", "dtype": "f32", "train": True, "rows": 4099, "q_heads": 9, "k_heads": 3, "head_dim": 80,
         "pairs": 20, "norm": "centred", "axes": 2, "layout": "neighbours", "start": 3},
        # A decoding step of 32 sequences: one new token each.
        {"name": "append_step_bf16", "op": "append", "dtype": "bf16", "kind": "plain", "documents": 32, "queries": 1, "past": 2048, "ragged": 4,
         "q_heads": 16, "kv_heads": 4, "head_dim": 128, "pairs": 64, "norm": "rms", "layout": "halves", "page": 64, "order": "heads"},
        # Chunks of four prompts into 4-bit pages.
        {"name": "append_chunks_int4_bf16", "op": "append", "dtype": "bf16", "kind": "int4", "documents": 4, "queries": 2048, "past": 300, "ragged": 0,
         "q_heads": 16, "kv_heads": 4, "head_dim": 128, "pairs": 64, "norm": "rms", "layout": "halves", "page": 64, "order": "heads"},
        # Five drafted tokens of each of seven sequences into 4-bit pages, tokens before heads, part of the head turned.
        {"name": "append_drafts_int4_f16", "op": "append", "dtype": "f16", "kind": "int4", "documents": 7, "queries": 5, "past": 77, "ragged": 2,
         "q_heads": 12, "kv_heads": 4, "head_dim": 96, "pairs": 24, "norm": "none", "layout": "neighbours", "page": 16, "order": "rows"},
        # Sixteen sequences decoded one token at a time over ragged pages.
        {"name": "decode_bf16", "op": "attention", "dtype": "bf16", "kind": "plain", "documents": 16, "queries": 1, "mixed": 0, "keys": 16384, "ragged": 3,
         "q_heads": 16, "kv_heads": 4, "head_dim": 128, "mask": "causal", "window": 0, "cap": 0.0, "page": 64, "order": "heads", "spare": 0},
        # Thirty-two sequences over pages of 4 bits, more key heads.
        {"name": "decode_int4_bf16", "op": "attention", "dtype": "bf16", "kind": "int4", "documents": 32, "queries": 1, "mixed": 0, "keys": 16384, "ragged": 5,
         "q_heads": 32, "kv_heads": 8, "head_dim": 128, "mask": "causal", "window": 0, "cap": 0.0, "page": 64, "order": "heads", "spare": 0},
        # One short sequence's next token over 4 bits: latency alone.
        {"name": "decode_one_int4_f16", "op": "attention", "dtype": "f16", "kind": "int4", "documents": 1, "queries": 1, "mixed": 0, "keys": 700, "ragged": 0,
         "q_heads": 12, "kv_heads": 12, "head_dim": 64, "mask": "causal", "window": 0, "cap": 0.0, "page": 32, "order": "heads", "spare": 0},
        # Drafted tokens checked over the nearest keys, tokens before heads in small pages.
        {"name": "drafts_window_f16", "op": "attention", "dtype": "f16", "kind": "plain", "documents": 9, "queries": 5, "mixed": 0, "keys": 6001, "ragged": 7,
         "q_heads": 24, "kv_heads": 3, "head_dim": 64, "mask": "causal", "window": 2049, "cap": 0.0, "page": 16, "order": "rows", "spare": 11},
        # Full precision with an odd head and odd lengths, scores capped.
        {"name": "drafts_odd_f32", "op": "attention", "dtype": "f32", "kind": "plain", "documents": 3, "queries": 3, "mixed": 0, "keys": 1777, "ragged": 2,
         "q_heads": 6, "kv_heads": 2, "head_dim": 40, "mask": "causal", "window": 0, "cap": 12.0, "page": 48, "order": "heads", "spare": 3},
        # A batch of prompts' chunks and single tokens together, scores capped.
        {"name": "chunks_cap_bf16", "op": "attention", "dtype": "bf16", "kind": "plain", "documents": 8, "queries": 1024, "mixed": 1, "keys": 8192, "ragged": 6,
         "q_heads": 16, "kv_heads": 4, "head_dim": 128, "mask": "causal", "window": 0, "cap": 30.0, "page": 64, "order": "heads", "spare": 5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["heads", "append", "attention"], [2, 2, 4])[0]
    dtype = rng.choice(["f32", "f16", "bf16"])
    layout = rng.choice(["halves", "neighbours"])
    if op == "heads":
        head_dim = 8 * rng.randint(2, 32)
        axes = rng.randint(1, 3)
        pairs = rng.choice([head_dim // 2, rng.randint(axes, head_dim // 2)])
        k_heads = rng.randint(1, 8)
        q_heads = k_heads * rng.randint(1, 6)
        rows = _log_int(rng, 1, 60_000_000 // (head_dim * (q_heads + k_heads)))
        return {"op": op, "dtype": dtype, "train": rng.random() < 0.6, "rows": rows, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim,
                "pairs": pairs, "norm": rng.choice(["rms", "centred"]), "axes": axes, "layout": layout,
                "start": rng.choice([0, _log_int(rng, 1, 2_000_000)])}
    kind = rng.choice(["plain", "int4"])
    head_dim = 8 * rng.randint(2, 16) if kind == "plain" else 32 * rng.randint(1, 4)
    kv_heads = rng.randint(1, 8)
    q_heads = kv_heads * rng.randint(1, 8)
    page, order = 16 * rng.choice([1, 2, 3, 4, 8]), rng.choice(["heads", "rows"])
    common = {"op": op, "dtype": dtype, "kind": kind, "documents": _log_int(rng, 1, 48), "ragged": rng.randint(0, 9), "q_heads": q_heads,
              "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "order": order}
    if op == "append":
        room = 8192 * 24 * 128 // ((q_heads + 2 * kv_heads) * head_dim * common["documents"])
        queries = rng.choice([1, rng.randint(2, 9), _log_int(rng, 1, max(2, min(4096, room)))])
        pairs = rng.choice([head_dim // 2, rng.randint(1, head_dim // 2)])
        return {**common, "queries": min(queries, max(1, room)), "past": _log_int(rng, 1, max(2, min(2000, room))), "pairs": pairs,
                "norm": rng.choice(["none", "rms", "centred"]), "layout": layout}
    common.update(mixed=rng.randint(0, 1), mask=rng.choice(["none", "causal", "causal"]), cap=rng.choice([0.0, 0.0, 15.0, 50.0]), spare=rng.choice([0, 0, 19]))
    # what the largest listed cache holds
    room = 32 * 16384 * 8 * 128 // (common["documents"] * kv_heads * head_dim)
    if rng.random() < 0.65:  # a few tokens over a cache
        queries = rng.choice([1, 1, 1, rng.randint(2, 9)])
        keys = _log_int(rng, 9, max(10, min(60_000, room // (3 * queries))))
    else:  # chunks of prompts: the plain form's scores, and less in f32
        pairs = 8 * 1024 * 8192 * 16 // ((8 if dtype == "f32" else 2) * common["documents"] * q_heads)
        queries = _log_int(rng, 10, max(11, min(2048, int(math.sqrt(pairs / 2)))))
        keys = min(queries * rng.randint(1, 8) + rng.randint(0, 99), max(queries, pairs // queries), 16384)
    window = rng.choice([0, 0, _log_int(rng, 1, keys)]) if common["mask"] == "causal" else 0
    return {**common, "queries": queries, "keys": max(keys, queries), "window": window}


# ---------------------------------------------------------------------------
# sizes that follow from a case alone
# ---------------------------------------------------------------------------


def _lengths(case):
    """(new tokens or queries, cached keys with them) of each document."""
    r = random.Random(case["ragged"])
    got = []
    for i in range(case["documents"]):
        f = 1.0 if case["ragged"] == 0 else r.uniform(0.2, 1.0)
        if case["op"] == "append":
            n = max(1, int(case["queries"] * f))
            got.append((n, n + int(case["past"] * f)))
        else:
            n = 1 if case["mixed"] and i % 2 else case["queries"]
            got.append((n, max(n, int(case["keys"] * f))))
    return got


def _pages(case):
    """(pages of each document, pages of the cache)."""
    of = [-(-n // case["page"]) for _, n in _lengths(case)]
    return of, sum(of) + 2


def _row_bytes(case):
    d = case["head_dim"]
    return d // 2 + d // 8 if case["kind"] == "int4" else d * (4 if case["dtype"] == "f32" else 2)


def _seen(case, n_q, n_k):
    """(query, key) pairs that the masks leave, and keys that some query sees."""
    if case["mask"] == "none":
        return n_q * n_k, n_k
    w = case["window"] or n_k
    return sum(min(w, n_k - n_q + i + 1) for i in range(n_q)), min(n_k, n_q + w - 1)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    d = case["head_dim"]
    if case["op"] == "heads":
        n = case["rows"] * (case["q_heads"] + case["k_heads"]) * d
        turned = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["pairs"]
        # forward x -> y; backward dy, x -> dx; positions, and the weights and their gradients
        once = 2 * n * size + 4 * case["rows"] * case["axes"] + 2 * d * size
        back = 3 * n * size + 4 * case["rows"] * case["axes"] + 2 * d * (size + 4)
        return {"bytes": once + (back if case["train"] else 0), "flops": (5 * n + 6 * turned) + ((12 * n + 6 * turned) if case["train"] else 0)}
    lens = _lengths(case)
    if case["op"] == "append":
        rows = sum(n for n, _ in lens)
        bytes_ = rows * (2 * case["q_heads"] + 2 * case["kv_heads"]) * d * size + 2 * rows * case["kv_heads"] * _row_bytes(case)
        if case["kind"] == "int4":  # the documents' values are read back
            keys = sum(n for _, n in lens) * case["kv_heads"] * 2
            bytes_ += keys * (_row_bytes(case) + 2 * d)
        return {"bytes": bytes_, "flops": rows * (case["q_heads"] + case["kv_heads"]) * (5 * d + 6 * case["pairs"]) + rows * case["kv_heads"] * d * 8}
    q = sum(n for n, _ in lens) * case["q_heads"]
    seen = [_seen(case, *n) for n in lens]
    bytes_ = 2 * q * d * size + 4 * q + 2 * sum(k for _, k in seen) * case["kv_heads"] * _row_bytes(case)
    return {"bytes": bytes_, "flops": 4.0 * sum(p for p, _ in seen) * case["q_heads"] * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device="cuda") * scale).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _grid_positions(n, axes, start=0):
    """Positions of n tokens: a text's, an image's rows and columns, or a
    video's frames of such images; [n][axes]."""
    t = torch.arange(n, device="cuda", dtype=torch.int32)
    if axes <= 1:
        return (t + start)[:, None]
    if axes == 2:
        w = max(1, math.isqrt(n))
        return torch.stack([t // w + start, t % w + start], 1)
    w = max(1, round(n ** (1 / 3)))
    return torch.stack([t // (w * w) + start, t // w % w + start, t % w + start], 1)


def _sections(case):
    axes, pairs = case.get("axes", 1), case["pairs"]
    return [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]


def _ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _prepare_cache(s, r):
    """A pool of pages in the case's order, every row of it filled by earlier
    steps, and dealt out at random."""
    case = s["case"]
    of, pages = _pages(case)
    heads, page, d = case["kv_heads"], case["page"], case["head_dim"]
    shape = (heads, page) if case["order"] == "heads" else (page, heads)
    for name in ("k_pages", "v_pages"):
        if case["kind"] == "plain":
            s[name] = r.normal(pages, *shape, d, dtype=DTYPES[case["dtype"]])
            continue
        s[name] = torch.empty(pages, *shape, d // 2 + d // 8, device="cuda", dtype=torch.uint8)
        step = max(1, (1 << 26) // (heads * page * d))  # a large pool some pages at a time
        for at in range(0, pages, step):
            n = min(step, pages - at)
            s[name][at:at + n] = _codes_of(r.normal(n, *shape, d))
    deal = r.order(pages).tolist()
    table, at = [], 0
    for n in of:
        table.append(deal[at:at + n] + [-1] * (max(of) - n))
        at += n
    s["table"] = _ints(table)
    s["lengths"] = _ints([n for _, n in _lengths(case)])


def prepare(case, seed):
    r, dtype = _Random(seed), DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    d = case["head_dim"]
    if case["op"] == "heads":
        rows, hq, hk = case["rows"], case["q_heads"], case["k_heads"]
        # q and k lie side by side in the projection's output, with v behind them
        s["qkv"] = (r.normal(rows, hq + 2 * hk, d) * (0.3 + r.normal(d).abs()) + 0.2 * r.normal(d)).to(dtype)
        s["q_gamma"], s["k_gamma"] = ((1.0 + 0.2 * r.normal(d)).to(dtype) for _ in range(2))
        s["positions"] = _grid_positions(rows, case["axes"], case["start"]).contiguous()
        s["q"], s["k"] = (torch.empty(rows, h, d, device="cuda", dtype=dtype) for h in (hq, hk))
        if case["train"]:
            s["d_q"], s["d_k"] = (r.normal(rows, h, d, dtype=dtype) for h in (hq, hk))
            s["d_qkv"] = torch.zeros(rows, hq + 2 * hk, d, device="cuda", dtype=dtype)
            s["d_q_gamma"], s["d_k_gamma"] = (torch.empty(d, device="cuda") for _ in range(2))
    else:
        hq, hk = case["q_heads"], case["kv_heads"]
        lens = _lengths(case)
        _prepare_cache(s, r)
        offsets = [0]
        for n, _ in lens:
            offsets.append(offsets[-1] + n)
        s["q_offsets"] = _ints(offsets)
        if case["op"] == "append":
            rows = offsets[-1]
            s["qkv"] = (r.normal(rows, hq + 2 * hk, d) * (0.7 + 0.3 * r.normal(d).abs())).to(dtype)
            s["q_gamma"], s["k_gamma"] = ((1.0 + 0.1 * r.normal(d)).to(dtype) for _ in range(2))
            s["q"] = torch.empty(rows, hq, d, device="cuda", dtype=dtype)
            if case["kind"] == "int4":  # the documents' values, read back
                first = [0]
                for _, n in lens:
                    first.append(first[-1] + n)
                s["key_offsets"] = _ints(first)
                s["k_values"], s["v_values"] = (torch.empty(first[-1], hk, d, device="cuda", dtype=torch.float16) for _ in range(2))
        else:
            rows = offsets[-1] + case["spare"]
            s["q"] = r.normal(rows, hq, d, scale=1.5, dtype=dtype)
            s["out"] = torch.zeros(rows, hq, d, device="cuda", dtype=dtype)
            s["lse"] = torch.zeros(hq, rows, device="cuda")
            s["scale"] = d ** -0.5
    if own:
        _prepare_calls(s)
    return s


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _prepare_calls(s):
    """The arguments a user's program keeps beside its buffers."""
    global _context
    from beatlm_amd import hip, ops

    if _context is None:
        _context = hip.Context(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream)
    case, ctx = s["case"], _context
    s["ctx"], s["ops"] = ctx, ops
    dtype = {"f32": hip.F32, "f16": hip.F16, "bf16": ops.BF16}[case["dtype"]]
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    heads = lambda t: ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    norm = {"none": ops.HEAD_NORM_NONE, "rms": ops.HEAD_NORM_RMS, "centred": ops.HEAD_NORM_CENTRED}
    d = case["head_dim"]

    def workspace(n):
        s["workspace"] = torch.empty(max(1, n), device="cuda", dtype=torch.uint8)
        return s["workspace"].data_ptr(), n

    def cache():
        def side(t):
            row, head = (2, 1) if case["order"] == "heads" else (1, 2)
            size = t.element_size()
            return ops.Pages(t.data_ptr(), t.stride(0) * size, t.stride(row) * size, t.stride(head) * size)
        return ops.PagedCache(kind=ops.CACHE_INT4 if case["kind"] == "int4" else ops.CACHE_PLAIN, pages=s["k_pages"].shape[0], page_rows=case["page"],
                              max_pages=s["table"].shape[1], table=at(s["table"]), lengths=at(s["lengths"]), k=side(s["k_pages"]), v=side(s["v_pages"]))

    if "pairs" in case:
        s["rotary"] = ops.rotary_table(_sections(case), BASE, neighbours=case["layout"] == "neighbours")
    if case["op"] == "heads":
        hq, hk = case["q_heads"], case["k_heads"]
        s["args"] = ops.HeadNormArgs(
            dtype=dtype, rows=case["rows"], q_heads=hq, k_heads=hk, head_dim=d, norm=norm[case["norm"]], epsilon=EPSILON, positions=at(s["positions"]),
            q_gamma=at(s["q_gamma"]), k_gamma=at(s["k_gamma"]), q_in=heads(s["qkv"][:, :hq]), k_in=heads(s["qkv"][:, hq:hq + hk]),
            q_out=heads(s["q"]), k_out=heads(s["k"]))
        if case["train"]:
            w, n = workspace(ops.head_norm_rotary_backward_workspace(ctx, s["args"]))
            s["grads"] = ops.HeadNormGrads(dq_out=heads(s["d_q"]), dk_out=heads(s["d_k"]), dq_in=heads(s["d_qkv"][:, :hq]), dk_in=heads(s["d_qkv"][:, hq:hq + hk]),
                                           d_q_gamma=at(s["d_q_gamma"]), d_k_gamma=at(s["d_k_gamma"]), workspace=w, workspace_bytes=n)
    elif case["op"] == "append":
        hq, hk = case["q_heads"], case["kv_heads"]
        s["args"] = ops.CacheAppendArgs(
            dtype=dtype, rows=s["qkv"].shape[0], documents=case["documents"], q_heads=hq, kv_heads=hk, head_dim=d, norm=norm[case["norm"]], epsilon=EPSILON,
            q_offsets=at(s["q_offsets"]), positions=None, q_gamma=at(s["q_gamma"]), k_gamma=at(s["k_gamma"]), q_in=heads(s["qkv"][:, :hq]),
            q_out=heads(s["q"]), k_in=heads(s["qkv"][:, hq:hq + hk]), v_in=heads(s["qkv"][:, hq + hk:]), cache=cache())
        if case["kind"] == "int4":
            s["read"] = ops.CacheReadArgs(dtype=hip.F16, rows=s["k_values"].shape[0], documents=case["documents"], kv_heads=hk, head_dim=d,
                                          offsets=at(s["key_offsets"]), first=None, k_out=heads(s["k_values"]), v_out=heads(s["v_values"]), cache=cache())
    else:
        a = ops.PagedAttentionArgs(
            dtype=dtype, q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=d, q_rows=s["q"].shape[0], documents=case["documents"],
            mask=ops.MASK_CAUSAL if case["mask"] == "causal" else ops.MASK_NONE, window=case["window"], max_keys=max(n for _, n in _lengths(case)),
            scale=s["scale"], softcap=case["cap"], q_offsets=at(s["q_offsets"]), q=heads(s["q"]), out=heads(s["out"]), lse=at(s["lse"]), cache=cache())
        a.workspace, a.workspace_bytes = workspace(ops.paged_attention_workspace(ctx, a))
        s["args"] = a


def _run_own(s):
    case, ctx, ops = s["case"], s["ctx"], s["ops"]
    if case["op"] == "heads":
        ops.head_norm_rotary(ctx, s["rotary"], s["args"])
        if not case["train"]:
            return {"q": s["q"], "k": s["k"]}
        ops.head_norm_rotary_backward(ctx, s["rotary"], s["args"], s["grads"])
        return {n: s[n] for n in ("q", "k", "d_qkv", "d_q_gamma", "d_k_gamma")}
    if case["op"] == "append":
        ops.cache_append(ctx, s["rotary"], s["args"])
        if case["kind"] == "plain":
            return {"q": s["q"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        ops.cache_read(ctx, s["read"])
        return {"q": s["q"], "k_values": s["k_values"], "v_values": s["v_values"]}
    ops.paged_attention(ctx, s["args"])
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _codes_of(x):
    """Rows of 4-bit codes and their steps and lows, for x [..., head_dim]; what
    lies next to a border is decided in 64 bits."""
    g = x.unflatten(-1, (-1, GROUP)).double()
    top, low = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    step, low = ((top - low) / 15).to(torch.float16), low.to(torch.float16)
    code = ((g - low.double()) / step.double()).nan_to_num(0.0).round().clamp(0, 15)
    nibble = torch.empty_like(code.flatten(-2).unflatten(-1, (-1, 8)), dtype=torch.uint8)
    nibble[..., NIBBLES] = code.flatten(-2).unflatten(-1, (-1, 8)).to(torch.uint8)
    codes = (nibble[..., 0::2] | nibble[..., 1::2] << 4).flatten(-2)
    params = torch.cat([step, low], -1).flatten(-2).view(torch.uint8)
    return torch.cat([codes, params], -1)


def _values_of(rows, d):
    """What rows of 4-bit codes stand for, f16 values in 32 bits."""
    codes, params = rows[..., :d // 2], rows[..., d // 2:].contiguous().view(torch.float16).float()
    nibble = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))[..., NIBBLES]
    step, low = params.unflatten(-1, (-1, 2)).unbind(-1)
    value = nibble.flatten(-2).unflatten(-1, (-1, GROUP)).float() * step[..., None] + low[..., None]
    return value.to(torch.float16).float().flatten(-2)


def _plain_turn(x, cos, sin, case):
    """x [rows][heads][head_dim], turned by (cos, sin) [rows][1][pairs]."""
    p = case["pairs"]
    if case["layout"] == "halves":
        a, b = x[..., :p], x[..., p:2 * p]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * p:]], -1)
    a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * p:]], -1)


def _plain_angles(positions, case):
    pairs, sections = case["pairs"], _sections(case)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda")
    freq = BASE ** -(torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    angle = positions.double()[:, axis] * freq
    return angle.cos()[:, None], angle.sin()[:, None]


def _plain_norm(x, norm):
    """(n, rstd) of each head."""
    if norm == "none":
        return x, None
    if norm == "centred":
        x = x - x.mean(-1, keepdim=True)
    rstd = ((x * x).mean(-1, keepdim=True) + EPSILON).rsqrt()
    return x * rstd, rstd


def _plain_heads(s):
    case, dtype = s["case"], s["qkv"].dtype
    hq, hk = case["q_heads"], case["k_heads"]
    cos, sin = _plain_angles(s["positions"], case)
    cos, sin = cos.float(), sin.float()
    got, d_x = {}, []
    for name, x in (("q", s["qkv"][:, :hq]), ("k", s["qkv"][:, hq:hq + hk])):
        gamma = s[name + "_gamma"].float()
        n, rstd = _plain_norm(x.float(), case["norm"])
        got[name] = _plain_turn(n * gamma, cos, sin, case).to(dtype)
        if case["train"]:
            dz = _plain_turn(s["d_" + name].float(), cos, -sin, case)
            got["d_%s_gamma" % name] = (dz * n).sum((0, 1))
            g = dz * gamma
            dx = g - n * (g * n).mean(-1, keepdim=True)
            if case["norm"] == "centred":
                dx = dx - g.mean(-1, keepdim=True)
            d_x.append(dx * rstd)
    if case["train"]:
        got["d_qkv"] = torch.cat(d_x + [torch.zeros_like(d_x[1])], 1).to(dtype)
        return {n: got[n] for n in ("q", "k", "d_qkv", "d_q_gamma", "d_k_gamma")}
    return got


def _document_rows(offsets, rows):
    """(document, index in it, whether it has one) of each packed row."""
    row = torch.arange(rows, device="cuda")
    doc = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    inside = doc < offsets.shape[0] - 1
    doc = doc.clamp(max=offsets.shape[0] - 2)
    return doc, row - offsets[doc], inside


def _plain_append(s):
    case, dtype = s["case"], s["qkv"].dtype
    hq, hk, page, d = case["q_heads"], case["kv_heads"], case["page"], case["head_dim"]
    offsets, lengths, table = s["q_offsets"].long(), s["lengths"].long(), s["table"].long()
    doc, i, _ = _document_rows(offsets, s["qkv"].shape[0])
    place = lengths[doc] - (offsets[doc + 1] - offsets[doc]) + i
    cos, sin = _plain_angles(place[:, None], case)
    weighed = lambda x, gamma: x if case["norm"] == "none" else x * gamma  # noqa: E731
    q = weighed(_plain_norm(s["qkv"][:, :hq].float(), case["norm"])[0], s["q_gamma"].float())
    got = {"q": _plain_turn(q, cos.float(), sin.float(), case).to(dtype)}
    k, v = s["qkv"][:, hq:hq + hk], s["qkv"][:, hq + hk:]
    if case["kind"] == "int4":  # next to a border 32 bits lose what matters
        k = weighed(_plain_norm(k.double(), case["norm"])[0], s["k_gamma"].double())
        k = _codes_of(_plain_turn(k, cos, sin, case).float())
        v = _codes_of(v.float())
    else:
        k = weighed(_plain_norm(k.float(), case["norm"])[0], s["k_gamma"].float())
        k = _plain_turn(k, cos.float(), sin.float(), case).to(dtype)
    at, row = table[doc, place // page], place % page
    for name, x in (("k_pages", k), ("v_pages", v)):
        if case["order"] == "heads":
            s[name][at, :, row] = x
        else:
            s[name][at, row] = x
        if case["kind"] == "plain":
            got[name] = s[name]
    if case["kind"] == "int4":
        first = s["key_offsets"].long()
        doc, j, _ = _document_rows(first, s["k_values"].shape[0])
        at, row = table[doc, j // page], j % page
        for name in ("k", "v"):
            pool = s[name + "_pages"]
            rows = pool[at, :, row] if case["order"] == "heads" else pool[at, row]
            got[name + "_values"] = _values_of(rows, d).to(torch.float16)
    return got


def _plain_attention(s):
    case, dtype = s["case"], s["q"].dtype
    hq, hk, d, page, cap = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["cap"]
    lens = _lengths(case)
    docs, most_q, most_k = len(lens), max(n for n, _ in lens), max(n for _, n in lens)
    offsets, n_k, table = s["q_offsets"].long(), s["lengths"].long(), s["table"].long()
    n_q = offsets[1:] - offsets[:-1]
    i, j = torch.arange(most_q, device="cuda"), torch.arange(most_k, device="cuda")
    q = s["q"][(offsets[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)].float()
    q = q.view(docs, most_q, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(docs, hk, -1, d)

    at, row = table[:, j // page].clamp(min=0), (j % page)[None].expand(docs, -1)

    def side(pool):
        x = pool[at, :, row] if case["order"] == "heads" else pool[at, row]
        return (_values_of(x, d) if case["kind"] == "int4" else x.float()).permute(0, 2, 1, 3).contiguous()

    score = q @ side(s["k_pages"]).transpose(-1, -2).contiguous() * s["scale"]
    if cap:
        score = cap * (score / cap).tanh()
    place = i[None, :, None] + (n_k - n_q)[:, None, None]
    seen = (j < n_k[:, None, None]).expand(docs, most_q, most_k)
    if case["mask"] == "causal":
        seen = seen & (j <= place)
        if case["window"]:
            seen = seen & (j > place - case["window"])
    hidden = ~seen[:, None, None].expand(docs, 1, hq // hk, most_q, most_k).reshape(docs, 1, -1, most_k)
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0]
    o = (p / total.clamp(min=1e-37)) @ side(s["v_pages"])
    # back to packed rows, those behind the last document as they were
    doc, index, inside = _document_rows(offsets, s["q"].shape[0])
    o = o.view(docs, hk, hq // hk, most_q, d).permute(0, 3, 1, 2, 4).reshape(docs, most_q, hq, d)[doc, index.clamp(max=most_q - 1)]
    lse = lse.view(docs, hq, most_q).permute(0, 2, 1)[doc, index.clamp(max=most_q - 1)]
    return {"out": o.masked_fill(~inside[:, None, None], 0.0).to(dtype), "lse": lse.masked_fill(~inside[:, None], 0.0).t().contiguous()}


def run(state):
    if own:
        return _run_own(state)
    return {"heads": _plain_heads, "append": _plain_append, "attention": _plain_attention}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_normed(x, gamma, norm):
    if norm == "none":
        return x
    if norm == "centred":
        x = x - x.sum(-1, keepdim=True) / x.shape[-1]
    return x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPSILON) * gamma


def _exact_phases(positions, case):
    """exp(i angle) of each row and pair."""
    turns, first = [], 0
    for axis, n in enumerate(_sections(case)):
        for i in range(first, first + n):
            angle = positions[:, axis].double() * math.exp(-i / case["pairs"] * math.log(BASE))
            turns.append(torch.polar(torch.ones_like(angle), angle))
        first += n
    return torch.stack(turns, 1)[:, None]


def _exact_turned(x, phase, case):
    p = case["pairs"]
    if case["layout"] == "halves":
        z = torch.complex(x[..., :p], x[..., p:2 * p]) * phase
        return torch.cat([z.real, z.imag, x[..., 2 * p:]], -1)
    z = torch.view_as_real(torch.complex(x[..., 0:2 * p:2], x[..., 1:2 * p:2]) * phase)
    return torch.cat([z.reshape(*x.shape[:-1], 2 * p), x[..., 2 * p:]], -1)


def _exact_heads(s):
    case = s["case"]
    hq, hk = case["q_heads"], case["k_heads"]
    phase = _exact_phases(s["positions"], case)
    got = {"d_qkv": torch.zeros(s["qkv"].shape, device="cuda", dtype=torch.float64)}
    for name, heads in (("q", slice(0, hq)), ("k", slice(hq, hq + hk))):
        x, gamma = s["qkv"][:, heads].double().requires_grad_(case["train"]), s[name + "_gamma"].double().requires_grad_(case["train"])
        y = _exact_turned(_exact_normed(x, gamma, case["norm"]), phase, case)
        got[name] = y.detach()
        if case["train"]:
            got["d_qkv"][:, heads], got["d_%s_gamma" % name] = torch.autograd.grad(y, (x, gamma), s["d_" + name].double())
    return {n: got[n] for n in (("q", "k", "d_qkv", "d_q_gamma", "d_k_gamma") if case["train"] else ("q", "k"))}


def _exact_code_values(x):
    """What the codes of x [..., 32 n] (f32) stand for."""
    got = torch.empty(x.shape, device="cuda", dtype=torch.float64)
    for c in range(0, x.shape[-1], GROUP):
        g = x[..., c:c + GROUP].double()
        low = g.min(-1, keepdim=True).values
        step = ((g.max(-1, keepdim=True).values - low) / 15.0).half().double()
        low = low.half().double()
        code = torch.where(step > 0, torch.round((g - low) / step.clamp(min=1e-30)), torch.zeros_like(g)).clamp(0, 15)
        got[..., c:c + GROUP] = (low + code * step).half().double()
    return got


def _exact_stored(rows, d):
    """What stored rows of codes stand for."""
    got = torch.empty(*rows.shape[:-1], d, device="cuda", dtype=torch.float64)
    words = rows[..., :d // 2].contiguous().view(torch.int32)
    params = rows[..., d // 2:].contiguous().view(torch.int16).view(torch.float16).double()
    for c in range(d):
        bits = (c % 8) // 2 * 4 + c % 2 * 16
        code = words[..., c // 8].bitwise_right_shift(bits) & 15
        got[..., c] = (params[..., c // GROUP * 2 + 1] + code.double() * params[..., c // GROUP * 2]).half().double()
    return got


def _exact_append(s):
    case = s["case"]
    hq, hk, page = case["q_heads"], case["kv_heads"], case["page"]
    lens, table = _lengths(case), s["table"].tolist()
    place = torch.cat([torch.arange(n_k - n_q, n_k, device="cuda") for n_q, n_k in lens])
    phase = _exact_phases(place[:, None], case)
    turned = lambda x, gamma: _exact_turned(_exact_normed(x.double(), gamma.double(), case["norm"]), phase, case)  # noqa: E731
    got = {"q": turned(s["qkv"][:, :hq], s["q_gamma"])}
    new = {"k": turned(s["qkv"][:, hq:hq + hk], s["k_gamma"]), "v": s["qkv"][:, hq + hk:].double()}
    for name, x in new.items():
        if case["kind"] == "int4":
            x = _exact_code_values(x.float())
        pool = s[name + "_pages"]
        pool = pool if case["order"] == "heads" else pool.transpose(1, 2)
        if case["kind"] == "plain":
            pool = pool.double()
        whole, first = [], 0
        for d, (n_q, n_k) in enumerate(lens):
            old = n_k - n_q
            if case["kind"] == "plain":
                for j in range(old, n_k):
                    pool[table[d][j // page], :, j % page] = x[first + j - old]
            else:
                if old:
                    at = torch.tensor(table[d][:-(-old // page)], device="cuda")
                    whole.append(_exact_stored(pool[at].transpose(1, 2).reshape(-1, hk, pool.shape[-1])[:old], case["head_dim"]))
                whole.append(x[first:first + n_q])
            first += n_q
        if case["kind"] == "plain":
            got[name + "_pages"] = pool if case["order"] == "heads" else pool.transpose(1, 2).contiguous()
        else:
            got[name + "_values"] = torch.cat(whole)
    return got


def _exact_attention(s):
    case = s["case"]
    hq, hk, d, page, cap = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["cap"]
    table, offsets = s["table"].tolist(), s["q_offsets"].tolist()
    out = torch.zeros(s["out"].shape, device="cuda", dtype=torch.float64)
    lse = torch.zeros(s["lse"].shape, device="cuda", dtype=torch.float64)
    for doc, (n_q, n_k) in enumerate(_lengths(case)):
        at = torch.tensor(table[doc][:-(-n_k // page)], device="cuda")
        keys = []
        for pool in (s["k_pages"], s["v_pages"]):
            x = pool[at] if case["order"] == "rows" else pool[at].transpose(1, 2)
            x = x.reshape(-1, hk, pool.shape[-1])[:n_k]
            keys.append(_exact_stored(x, d) if case["kind"] == "int4" else x.double())
        place = torch.arange(n_k - n_q, n_k, device="cuda")[:, None]
        key = torch.arange(n_k, device="cuda")[None]
        hidden = torch.zeros(n_q, n_k, device="cuda", dtype=torch.bool)
        if case["mask"] == "causal":
            hidden = key > place
            if case["window"]:
                hidden = hidden | (key <= place - case["window"])
        rows = slice(offsets[doc], offsets[doc + 1])
        for h in range(hq):
            x = (s["q"][rows, h].double() @ keys[0][:, h // (hq // hk)].T) * s["scale"]
            if cap:
                x = cap * torch.tanh(x / cap)
            x = x.masked_fill(hidden, -math.inf)
            lse[h, rows] = torch.logsumexp(x, 1)
            out[rows, h] = torch.softmax(x, 1) @ keys[1][:, h // (hq // hk)]
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    return {"heads": _exact_heads, "append": _exact_append, "attention": _exact_attention}[case["op"]](s)
