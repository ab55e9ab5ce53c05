"""What the heads' norms and the paged cache's calls write beside what else they
touch: indices, weights, statistics and workspaces that lie in a tensor or in a
page's rows are refused, those in the gaps between rows are not."""

import random

import pytest

from beatlm_amd import ops
from tests.test_sublayer_cache import (AT, INVALID, accepted, append_args, attention_args, cache, host, norm_args, norm_grads, read_args, refused,  # noqa: F401
                                       table)


@pytest.mark.parametrize("changed,says", [
    (dict(positions=3 * AT), "q_out is positions"), (dict(positions=3 * AT - 4), "q_out overlaps positions"), (dict(positions=5 * AT + 8), "k_out overlaps positions"),
])
def test_head_norm(host, changed, says):  # noqa: F811
    refused(host, "bl_head_norm_rotary", [table(), norm_args(**changed)], INVALID, says)
    accepted(host, "bl_head_norm_rotary", [None, norm_args(**changed)])  # positions are not read
    accepted(host, "bl_head_norm_rotary", [table(), norm_args(positions=3 * AT - 9 * 4)])  # they end where q_out begins


@pytest.mark.parametrize("changed,more,says", [
    (dict(positions=8 * AT), {}, "dq_in is positions"), (dict(positions=9 * AT + 4), {}, "dk_in overlaps positions"),
    ({}, dict(d_q_gamma=2 * AT), "d_q_gamma is q_in"), ({}, dict(d_q_gamma=8 * AT + 64), "d_q_gamma overlaps dq_in"), ({}, dict(d_k_gamma=7 * AT), "d_k_gamma is dk_out"),
    ({}, dict(d_k_gamma=9 * AT - 252), "d_k_gamma overlaps dk_in"), ({}, dict(workspace=6 * AT), "the workspace is dq_out"), ({}, dict(workspace=4 * AT), "the workspace is k_in"),
    ({}, dict(workspace=8 * AT - 16), "the workspace overlaps dq_in"),
])
def test_head_norm_backward(host, changed, more, says):  # noqa: F811
    refused(host, "bl_head_norm_rotary_backward", [table(), norm_args(**changed), norm_grads(**more)], INVALID, says)


def test_head_norm_backward_accepts_what_it_does_not_write(host):  # noqa: F811
    # 9 rows: 9 groups of 2 * 64 floats, and a workspace that is larger than the call needs
    accepted(host, "bl_head_norm_rotary_backward", [table(), norm_args(), norm_grads(workspace=8 * AT - 9 * 512, workspace_bytes=1 << 30)])
    accepted(host, "bl_head_norm_rotary_backward", [table(), norm_args(k_heads=0), norm_grads(d_k_gamma=8 * AT)])  # no heads, no gradient


@pytest.mark.parametrize("changed,says", [
    (dict(q_offsets=3 * AT), "q_out is q_offsets"), (dict(cache__table=3 * AT + 64), "q_out overlaps the cache's table"), (dict(cache__lengths=3 * AT - 8), "q_out overlaps the cache's lengths"),
    (dict(positions=3 * AT), "q_out is positions"), (dict(q_gamma=20 * AT), "q_gamma overlaps the cache's keys"), (dict(k_gamma=21 * AT + 256), "k_gamma overlaps the cache's values"),
    (dict(positions=20 * AT), "positions overlaps the cache's keys"), (dict(q_offsets=21 * AT), "q_offsets overlaps the cache's values"),
    (dict(cache__table=20 * AT - 56), "table overlaps the cache's keys"), (dict(cache__lengths=21 * AT + 9 * 4096 + 4092), "lengths overlaps the cache's values"),
])
def test_append(host, changed, says):  # noqa: F811
    refused(host, "bl_cache_append", [table(), append_args(**changed)], INVALID, says)


def test_append_accepts_what_lies_between_rows(host):  # noqa: F811
    # Rows of 128 bytes every 256, two heads 4096 apart in pages of 8704 bytes.
    wide = dict(cache__k=ops.Pages(20 * AT, 8704, 256, 4096), cache__v=ops.Pages(21 * AT, 8704, 256, 4096))
    for at in (20 * AT + 128, 20 * AT + 8704 - 512, 20 * AT + 3 * 8704 + 5 * 256 + 128):
        accepted(host, "bl_cache_append", [table(), append_args(k_gamma=at, q_offsets=at, cache__lengths=at, **wide)])
        refused(host, "bl_cache_append", [table(), append_args(k_gamma=at - 2, **wide)] if at != 20 * AT + 8704 - 512 else [table(), append_args(k_gamma=at - 256, **wide)],
                INVALID, "k_gamma overlaps the cache's keys")
    accepted(host, "bl_cache_append", [table(), append_args(q_gamma=20 * AT, norm=0)])  # not read
    accepted(host, "bl_cache_append", [None, append_args(positions=20 * AT)])
    accepted(host, "bl_cache_append", [table(), append_args(cache__table=20 * AT - 3 * 5 * 4)])  # ends where the pages begin


@pytest.mark.parametrize("changed,says", [
    (dict(offsets=4 * AT), "k_out is offsets"), (dict(first=5 * AT + 4), "v_out overlaps first"), (dict(cache__table=4 * AT - 4), "k_out overlaps the cache's table"),
    (dict(cache__lengths=5 * AT), "v_out is the cache's lengths"),
])
def test_read(host, changed, says):  # noqa: F811
    refused(host, "bl_cache_read", [read_args(**changed)], INVALID, says)


@pytest.mark.parametrize("changed,says", [
    (dict(q_offsets=3 * AT), "out is q_offsets"), (dict(cache__table=3 * AT + 4), "out overlaps the cache's table"), (dict(cache__lengths=3 * AT + 4), "out overlaps the cache's lengths"),
    (dict(lse=2 * AT), "lse is q"), (dict(lse=3 * AT - 4), "lse overlaps out"), (dict(lse=20 * AT + 64), "lse overlaps the cache's keys"),
    (dict(workspace=2 * AT), "the workspace is q"), (dict(workspace=3 * AT - 16), "the workspace overlaps out"), (dict(workspace=21 * AT), "the workspace overlaps the cache's values"),
])
def test_attention(host, changed, says):  # noqa: F811
    refused(host, "bl_paged_attention", [attention_args(cache__max_pages=500, **changed)], INVALID, says)


def test_attention_accepts_what_it_does_not_write(host):  # noqa: F811
    n = ops._U64()
    sizes = attention_args(cache__max_pages=500)
    assert host.bl_paged_attention_workspace(host.stand_in_ctx(), sizes, n) == 0 and n.value
    accepted(host, "bl_paged_attention", [attention_args(cache__max_pages=500, workspace=3 * AT - n.value, workspace_bytes=1 << 40)])
    accepted(host, "bl_paged_attention", [attention_args(cache__max_pages=1, workspace=3 * AT, lse=3 * AT - 9 * 4 * 4)])  # one workgroup a document: no workspace


@pytest.mark.parametrize("seed", range(300))
def test_blocks_beside_pages_of_any_strides(host, seed):  # noqa: F811
    """Weights at any place within and around the pages, against every row's bytes."""
    r = random.Random(seed)
    pages, heads, d = r.randint(1, 4), r.randint(1, 3), 8
    width, block = d * 2, r.choice([8, 16, 24]) * 2
    steps = {}
    extent = width
    for name in r.sample(["page", "row", "head"], 3):
        count = {"page": pages, "row": 16, "head": heads}[name]
        steps[name] = (extent + 15) // 16 * 16 + 16 * r.randint(0, 3)
        extent += steps[name] * (count - 1)
    at = 20 * AT + r.randint(-block, extent) // 2 * 2
    starts = [20 * AT + p * steps["page"] + n * steps["row"] + h * steps["head"] for p in range(pages) for n in range(16) for h in range(heads)]
    side = lambda base: ops.Pages(base, steps["page"], steps["row"], steps["head"])  # noqa: E731
    # An index array's bytes are the block: offsets of block / 4 - 1 documents.
    a = append_args(head_dim=d, kv_heads=heads, documents=block // 4 - 1, q_heads=0, q_in=ops.Heads(), q_out=ops.Heads(), norm=0,
                    cache=cache(pages=pages, k=side(20 * AT), v=side(40 * AT)), q_offsets=at // 4 * 4)
    a.k_in.row_stride = a.v_in.row_stride = heads * 64
    at = at // 4 * 4
    if any(s < at + block and at < s + width for s in starts):
        refused(host, "bl_cache_append", [None, a], INVALID, "q_offsets overlaps the cache's keys")
    else:
        accepted(host, "bl_cache_append", [None, a])
