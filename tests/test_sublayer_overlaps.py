"""What the packed sublayer's operators write lies apart from what else they
touch: overlaps that begin inside a tensor are refused, views that share an
address range without an element are not. The host side as it is, over
stand-ins; no GPU."""

import ctypes as C
import random

import pytest

from beatlm_amd import hip, ops
from tests.test_sublayer_ops import AT, INVALID, accepted, attention_args, attention_grads, host, norm_args, norm_grads, refused, rotary_args, table  # noqa: F401

ROW = 256 * 2  # bytes of a row of the stand-in attention's tensors: 4 heads of 64, bf16


@pytest.mark.parametrize("changed,says", [
    (dict(out=ops.Heads(AT + ROW, 256, 64)), "out overlaps q"),          # one row in
    (dict(out=ops.Heads(AT - 9 * ROW, 256, 64)), "out overlaps q"),      # its last row is q's first
    (dict(out=ops.Heads(AT + 128, 256, 64)), "out overlaps q"),          # one head in
    (dict(out=ops.Heads(AT + 9 * ROW + 384, 512, 64)), "out overlaps q"),  # q's last head of its last row, other strides
    (dict(k=ops.Heads(2 * AT + 16, 128, 64)), "out overlaps k"),
    (dict(v=ops.Heads(2 * AT + 9 * ROW + 496, 128, 64)), "out overlaps v"),  # out's last 16 bytes
    (dict(v=ops.Heads(2 * AT + 16, 0, 0)), "out overlaps v"),            # one row for all keys
    (dict(q=ops.Heads(2 * AT - 9 * ROW - 1024, 320, 64)), "out overlaps q"),
])
def test_an_output_that_begins_inside_an_input(host, changed, says):  # noqa: F811
    refused(host, host.bl_packed_attention, [attention_args(**changed)], INVALID, says)


@pytest.mark.parametrize("more,says", [
    (dict(d_q=ops.Heads(AT + ROW, 256, 64)), "d_q overlaps q"), (dict(d_k=ops.Heads(AT + 256, 256, 64)), "d_k overlaps q"),
    (dict(d_v=ops.Heads(3 * AT + 128, 128, 64)), "d_v overlaps d_k"), (dict(d_out=ops.Heads(4 * AT + 16, 256, 64)), "d_v overlaps d_out"),
    (dict(d_q=ops.Heads(2 * AT + 9 * ROW, 256, 64)), "d_q overlaps out"), (dict(d_v=ops.Heads(5 * AT + 384, 128, 64)), "d_v overlaps d_q"),
])
def test_gradients_that_begin_inside_a_tensor(host, more, says):  # noqa: F811
    refused(host, host.bl_packed_attention_backward, [attention_args(), attention_grads(**more)], INVALID, says)


def test_views_of_one_tensor_pass(host):  # noqa: F811
    """Four tensors side by side in each row; heads before rows; a row a tensor."""
    at = lambda heads: ops.Heads(AT + heads * 128, 768, 64)  # noqa: E731
    a = attention_args(q=at(0), k=at(4), v=at(6), out=at(8))
    accepted(host, host.bl_packed_attention, [a])
    grad = lambda heads: ops.Heads(8 * AT + heads * 128, 768, 64)  # noqa: E731
    accepted(host, host.bl_packed_attention_backward, [a, attention_grads(d_out=at(0), d_q=grad(0), d_k=grad(4), d_v=grad(6))])
    by_heads = lambda heads: ops.Heads(AT + heads * 20 * 128, 64, 20 * 64)  # noqa: E731
    accepted(host, host.bl_packed_attention, [attention_args(q=by_heads(0), k=by_heads(4), v=by_heads(6), out=by_heads(8))])
    accepted(host, host.bl_packed_attention, [attention_args(out=ops.Heads(AT + 20 * ROW, 256, 64))])  # right behind the keys


def elements(h, rows, heads, d, size):
    return {h.data + (r * h.row_stride + n * h.head_stride) * size + b for r in range(rows) for n in range(heads) for b in range(0, d * size, 16)}


def test_overlaps_against_every_element(host):  # noqa: F811
    rng, seen = random.Random(7), {True: 0, False: 0}
    for _ in range(6000):
        kv_heads = rng.choice([1, 2, 3])
        q_heads = kv_heads * rng.choice([1, 2])
        rows, k_rows, d = rng.randint(1, 6), rng.randint(1, 6), rng.choice([8, 16, 24])

        def view():
            small = lambda: 8 * rng.randint(0, 12)  # noqa: E731
            return ops.Heads(AT + 16 * rng.randint(0, 60), rng.choice([small(), 48 * rng.randint(0, 4)]), rng.choice([small(), d, 48 * rng.randint(0, 4)]))

        a = attention_args(q_heads=q_heads, kv_heads=kv_heads, head_dim=d, q_rows=rows, k_rows=k_rows, q=view(), k=view(), v=view(), out=view())
        ctx = host.stand_in_ctx()
        rc = host.bl_packed_attention(ctx, C.byref(a))
        said = host.stand_in_error().decode()
        if rc != hip.OK and "heads of" in said:
            continue  # out overlaps itself
        out = elements(a.out, rows, q_heads, d, 2)
        want = bool(out & elements(a.q, rows, q_heads, d, 2) or out & elements(a.k, k_rows, kv_heads, d, 2) or out & elements(a.v, k_rows, kv_heads, d, 2))
        assert (rc != hip.OK) == want, (said, want, [(h.data - AT, h.row_stride, h.head_stride) for h in (a.q, a.k, a.v, a.out)], rows, k_rows, q_heads, kv_heads, d)
        seen[want] += 1
    assert min(seen.values()) > 200, seen


def test_overlaps_of_many_rows_against_every_element(host):  # noqa: F811
    rng, seen = random.Random(8), {True: 0, False: 0}
    for _ in range(4000):
        rows, cols = rng.randint(1, 200), rng.randint(1, 4)
        a = norm_args(rows=rows, cols=cols, x_stride=rng.randint(cols, 60), y_stride=rng.randint(cols, 60), x=AT, gamma=9 * AT, beta=9 * AT)
        if rng.random() < 0.5:  # rows that keep missing each other, by steps of one pitch
            pitch = rng.choice([6, 8, 12])
            a.x_stride, a.y_stride = pitch * rng.randint(1, 6), pitch * rng.randint(1, 6)
        a.y = AT + 2 * rng.randint(-1500, 1500)
        if a.y == AT:
            continue
        x, y = ({at + 2 * (r * stride + c) for r in range(rows) for c in range(cols)} for at, stride in ((a.x, a.x_stride), (a.y, a.y_stride)))
        rc = host.bl_layer_norm(host.stand_in_ctx(), C.byref(a))
        want = bool(x & y)
        assert (rc != hip.OK) == want, (host.stand_in_error(), want, rows, cols, a.x_stride, a.y_stride, a.y - AT)
        seen[want] += 1
    assert min(seen.values()) > 500, seen


@pytest.mark.parametrize("changed,says", [
    (dict(y=AT + 2), "y overlaps x"), (dict(y=AT + 40, y_stride=20), "y overlaps x"), (dict(x=2 * AT + 3 * 48 + 38), "y overlaps x"),
    (dict(gamma=2 * AT + 10), "y overlaps gamma"), (dict(beta=2 * AT + 48 - 10 + 20), "y overlaps beta"),
])
def test_a_layer_norm_over_part_of_its_input(host, changed, says):  # noqa: F811
    refused(host, host.bl_layer_norm, [norm_args(**changed)], INVALID, says)


@pytest.mark.parametrize("more,says", [
    (dict(dx=AT + 2), "dx overlaps"), (dict(dy=3 * AT + 40), "dx overlaps dy"), (dict(dx=AT + 40, dx_stride=24), "dx overlaps x"),
])
def test_layer_norm_gradients_over_part_of_an_input(host, more, says):  # noqa: F811
    refused(host, host.bl_layer_norm_backward, [norm_args(gamma=9 * AT), norm_grads(**more)], INVALID, says)


def test_layer_norms_side_by_side_pass(host):  # noqa: F811
    accepted(host, host.bl_layer_norm, [norm_args(x_stride=40, y=AT + 40, y_stride=40, gamma=5 * AT, beta=5 * AT)])
    accepted(host, host.bl_layer_norm, [norm_args(y=AT, y_stride=20, gamma=5 * AT, beta=5 * AT)])
    accepted(host, host.bl_layer_norm_backward, [norm_args(x_stride=60), norm_grads(dx=AT + 80, dx_stride=60, dy_stride=60, dy=AT + 40)])
    accepted(host, host.bl_layer_norm_backward, [norm_args(gamma=5 * AT), norm_grads(dx=AT)])


@pytest.mark.parametrize("changed,says", [
    (dict(q_out=ops.Heads(AT + 4, 256, 64)), "q_out overlaps q_in"), (dict(k_out=ops.Heads(2 * AT + 256, 256, 64)), "k_out overlaps q_out"),
    (dict(k_out=ops.Heads(2 * AT, 256, 64)), "k_out is q_out"), (dict(k_in=ops.Heads(3 * AT + 1024, 256, 64)), "k_out overlaps k_in"),
    (dict(k_in=ops.Heads(2 * AT + 512, 256, 64)), "q_out overlaps k_in"), (dict(q_in=ops.Heads(3 * AT + 256, 256, 64)), "k_out overlaps q_in"),
])
def test_rotary_outputs_over_part_of_another(host, changed, says):  # noqa: F811
    refused(host, host.bl_rotary, [table(), rotary_args(**changed)], INVALID, says)


def test_rotary_views_of_one_tensor_pass(host):  # noqa: F811
    at = lambda heads: ops.Heads(AT + heads * 256, 512, 64)  # noqa: E731
    accepted(host, host.bl_rotary, [table(), rotary_args(q_in=at(0), q_out=at(0), k_in=at(4), k_out=at(4))])
    accepted(host, host.bl_rotary, [table(), rotary_args(q_in=at(0), q_out=at(6 - 6), k_in=at(4), k_out=at(6))])
