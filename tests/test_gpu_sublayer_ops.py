"""LayerNorm, rotary positions and packed attention (beatlm_amd.ops) against
their formulas in 64 bits: types, head layouts, lengths, strides and masks
where they can go wrong, gradients against the formulas and against
differences, graphs, streams, and the operators run together."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.opsdata import DTYPES, F32, Packed, assert_within, half_step

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
# LayerNorm
# ---------------------------------------------------------------------------


class Norm:
    def __init__(self, rows, cols, dtype, stride=None, seed=1, offset=0.5):
        self.torch_dtype, self.dtype = DTYPES[dtype]
        self.rows, self.cols, self.stride = rows, cols, stride or cols
        g = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: torch.randn(*s, generator=g, device="cuda").to(self.torch_dtype)  # noqa: E731
        self.x, self.dy = make(rows, self.stride) + offset, make(rows, self.stride)
        self.gamma, self.beta = make(cols) * 0.3 + 1, make(cols)
        self.y, self.dx = (torch.full_like(self.x, 7.0) for _ in range(2))
        self.mean, self.rstd = (torch.full((rows,), 7.0, device="cuda") for _ in range(2))
        self.d_gamma, self.d_beta = (torch.full((cols,), 7.0, device="cuda") for _ in range(2))

    def args(self):
        return ops.LayerNormArgs(dtype=self.dtype, rows=self.rows, cols=self.cols, epsilon=1e-5, x_stride=self.stride, y_stride=self.stride,
                                 x=self.x.data_ptr(), gamma=self.gamma.data_ptr(), beta=self.beta.data_ptr(), y=self.y.data_ptr(),
                                 mean=self.mean.data_ptr(), rstd=self.rstd.data_ptr())

    def grads(self, ctx):
        n = ops.layer_norm_backward_workspace(ctx, self.args())
        self.workspace = torch.full((n + 16,), 0xFF, device="cuda", dtype=torch.uint8)
        return ops.LayerNormGrads(dy=self.dy.data_ptr(), dy_stride=self.stride, dx=self.dx.data_ptr(), dx_stride=self.stride,
                                  d_gamma=self.d_gamma.data_ptr(), d_beta=self.d_beta.data_ptr(), workspace=self.workspace.data_ptr(),
                                  workspace_bytes=n)

    def check(self):
        u, c = half_step(self.torch_dtype), self.cols
        tiny = 2.0**-25 if self.torch_dtype == torch.float16 else 1e-37
        x, dy = self.x[:, :c].double(), self.dy[:, :c].double()
        gamma, beta = self.gamma.double(), self.beta.double()
        mean = x.mean(1, keepdim=True)
        variance = ((x - mean) ** 2).mean(1, keepdim=True)
        rstd = (variance + 1e-5).rsqrt()
        n = (x - mean) * rstd
        # A row's sum: 16 values a thread, then at most 6 + 16 additions.
        sums = F32 * 40
        mean_off = sums * x.abs().mean(1, keepdim=True) + F32 * mean.abs()
        rstd_off = rstd * (sums + 8 * F32 + 2 * mean_off * rstd)
        n_off = mean_off * rstd + n.abs() * (rstd_off / rstd + 2 * F32) + F32 * x.abs() * rstd
        assert_within(self.mean, mean[:, 0], mean_off[:, 0], "mean")
        assert_within(self.rstd, rstd[:, 0], rstd_off[:, 0], "rstd")
        y = n * gamma + beta
        assert_within(self.y[:, :c], y, u * y.abs() + n_off * gamma.abs() + 3 * F32 * (n * gamma).abs() + 3 * F32 * beta.abs() + tiny, "y")
        assert torch.all(self.y[:, c:] == 7.0)
        g = dy * gamma
        m0, m1 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
        dx = rstd * (g - m0 - n * m1)
        size = (g.abs() + g.abs().mean(1, keepdim=True) + n.abs() * (g * n).abs().mean(1, keepdim=True)) * rstd
        spread = rstd * (n_off * m1.abs() + n.abs() * (g.abs() * n_off).mean(1, keepdim=True))
        assert_within(self.dx[:, :c], dx, u * dx.abs() + (sums + 8 * F32) * size + dx.abs() * rstd_off / rstd + spread + tiny, "dx")
        assert torch.all(self.dx[:, c:] == 7.0)
        rows = F32 * (self.rows + 8)
        assert_within(self.d_beta, dy.sum(0), rows * dy.abs().sum(0), "d_beta")
        assert_within(self.d_gamma, (dy * n).sum(0), rows * (dy * n).abs().sum(0) + (dy.abs() * n_off).sum(0) + 1e-30, "d_gamma")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols,stride", [
    (1, 1, None), (1, 8, None), (3, 7, None), (5, 384, None), (1370, 384, 400), (257, 513, None), (2, 1000, None), (9, 1024, 1032),
    (700, 768, None), (4, 1025, None), (33, 4096, None), (3, 4097, None), (2, 16384, None), (5, 12288, 12290), (1, 4096, None), (2050, 64, 66),
])
def test_layer_norm_and_its_gradients(gpu, dtype, rows, cols, stride):
    t = Norm(rows, cols, dtype, stride)
    ops.layer_norm(gpu, t.args())
    ops.layer_norm_backward(gpu, t.args(), t.grads(gpu))
    t.check()


def test_layer_norm_of_a_large_offset_keeps_its_variance(gpu):
    t = Norm(64, 768, "f32", offset=3000.0)
    ops.layer_norm(gpu, t.args())
    ops.layer_norm_backward(gpu, t.args(), t.grads(gpu))
    t.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_in_place_unaligned_and_without_statistics(gpu, dtype):
    t, w = Norm(37, 640, dtype), Norm(37, 640, dtype)
    ops.layer_norm(gpu, w.args())
    ops.layer_norm_backward(gpu, w.args(), w.grads(gpu))
    a = t.args()
    a.y, a.mean, a.rstd = t.x.data_ptr(), None, None
    flat = torch.zeros(37 * 640 + 1, device="cuda", dtype=t.torch_dtype)
    flat[1:] = t.x.flatten()
    ops.layer_norm(gpu, a)
    assert torch.equal(t.x, w.y)
    b = w.args()
    b.x = b.y = flat[1:].data_ptr()  # one element off every 16-byte boundary, in place
    ops.layer_norm(gpu, b)
    assert_within(flat[1:].view(37, 640), w.y.double(), (2 * half_step(t.torch_dtype) + 64 * F32) * (w.y.double().abs() + 1), "unaligned")
    for source in ("x", "dy"):  # dx over x, and over dy
        s = Norm(37, 640, dtype)
        ops.layer_norm(gpu, s.args())
        g = s.grads(gpu)
        g.dx = getattr(s, source).data_ptr()
        ops.layer_norm_backward(gpu, s.args(), g)
        assert torch.equal(getattr(s, source), w.dx)


def test_layer_norm_of_no_rows_clears_the_weights_gradients(gpu):
    t = Norm(1, 40, "f32")
    a = t.args()
    a.rows = 0
    ops.layer_norm(gpu, a)
    g = t.grads(gpu)
    ops.layer_norm_backward(gpu, a, g)
    assert torch.all(t.d_gamma == 0) and torch.all(t.d_beta == 0) and torch.all(t.y == 7) and torch.all(t.dx == 7)


def test_layer_norm_gradients_repeat_bit_for_bit(gpu):
    t = Norm(5000, 384, "bf16")
    ops.layer_norm(gpu, t.args())
    g = t.grads(gpu)
    ops.layer_norm_backward(gpu, t.args(), g)
    first = t.d_gamma.clone(), t.d_beta.clone(), t.dx.clone()
    for _ in range(3):
        ops.layer_norm_backward(gpu, t.args(), g)
        assert all(torch.equal(a, b) for a, b in zip(first, (t.d_gamma, t.d_beta, t.dx)))


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def rotary_reference(x, positions, table, inverse):
    """In 64 bits, from the table's own revolutions."""
    p = table.pairs
    axis = torch.tensor(list(table.axis[:p]), device="cuda", dtype=torch.long)
    turns = torch.tensor(list(table.turns[:p]), device="cuda", dtype=torch.float64)
    phi = (positions.double()[:, axis] * turns * (2 * math.pi))[:, None]
    c, s = phi.cos(), phi.sin() * (-1 if inverse else 1)
    x = x.double()
    y, size = x.clone(), x.abs().clone()
    first, second = (slice(0, p), slice(p, 2 * p)) if table.layout == ops.ROTARY_HALVES else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size[..., first] = size[..., second] = a.abs() + b.abs()
    return y, size


def rotary_check(got, x, positions, table, inverse, what):
    want, size = rotary_reference(x, positions, table, inverse)
    u = half_step(got.dtype)
    tiny = 2.0**-25 if got.dtype == torch.float16 else 1e-38
    # a sine of f32 (a few steps of 1), the fraction's rounding times 2 pi, two products and a sum;
    # the reference's own angle in 64 bits, whose rounding grows with it
    angle = 2 * math.pi * float(positions.abs().max() if positions.numel() else 0) * 2.0**-51
    assert_within(got, want, u * want.abs() + (16 * F32 + angle) * size + tiny, what)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,q_heads,k_heads,d,sections,per_axis,neighbours,start", [
    (1, 1, 1, 8, [4], False, False, 0),
    (1370, 6, 6, 64, [16, 16], True, False, 0),
    (1000, 16, 4, 128, [16, 24, 24], False, False, 7),
    (5, 9, 3, 80, [20], False, True, 1000003),
    (33, 3, 0, 24, [3, 4], False, False, 12),       # odd pairs: channel by channel; no key heads
    (33, 0, 2, 40, [8, 8], True, True, 3),
    (257, 2, 1, 256, [128], False, True, 2**31 - 300),
    (64, 5, 1, 256, [1], False, False, 5),          # one pair, a long tail
    (4099, 1, 1, 20, [3, 1, 4], True, True, 0),
])
@pytest.mark.parametrize("inverse", [0, 1])
def test_rotary_positions(gpu, dtype, rows, q_heads, k_heads, d, sections, per_axis, neighbours, start, inverse):
    torch_dtype, code = DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    heads = q_heads + k_heads
    qkv = torch.randn(rows, heads + 1, d, generator=g, device="cuda").to(torch_dtype)
    q, k = qkv[:, :q_heads], qkv[:, q_heads:heads]
    positions = (torch.arange(rows, device="cuda")[:, None] * torch.tensor([1, -2, 3], device="cuda")[: len(sections)] + start)
    positions = positions.clamp(-2**31, 2**31 - 1).to(torch.int32).contiguous()
    table = ops.rotary_table(sections, 10000.0, per_axis, neighbours)
    out = torch.full((rows, heads + 2, d), 7.0, device="cuda", dtype=torch_dtype)
    q_out, k_out = out[:, :q_heads], out[:, q_heads + 1:heads + 1]
    view = lambda t: ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    a = ops.RotaryArgs(dtype=code, rows=rows, q_heads=q_heads, k_heads=k_heads, head_dim=d, inverse=inverse, positions=positions.data_ptr(),
                       q_in=view(q), q_out=view(q_out), k_in=view(k), k_out=view(k_out))
    ops.rotary(gpu, table, a)
    rotary_check(q_out, q, positions, table, inverse, "q")
    rotary_check(k_out, k, positions, table, inverse, "k")
    assert torch.all(out[:, q_heads] == 7.0) and torch.all(out[:, heads + 1] == 7.0)
    want = out.clone()
    a.q_out, a.k_out = a.q_in, a.k_in  # in place: the same bits
    ops.rotary(gpu, table, a)
    assert torch.equal(q, want[:, :q_heads]) and torch.equal(k, want[:, q_heads + 1:heads + 1])


def test_rotary_by_a_table_of_the_host_s_own(gpu):
    """Frequencies and an order of axes that no ladder makes."""
    t = ops.RotaryTable(axes=2, pairs=8, layout=ops.ROTARY_HALVES)
    for i in range(8):
        t.turns[i], t.axis[i] = 0.01 * (i + 1) ** 2 - 0.3, i % 2
    x = torch.randn(50, 2, 16, device="cuda")
    y = torch.empty_like(x)
    positions = torch.randint(-1000, 1000, (50, 2), device="cuda", dtype=torch.int32)
    view = lambda v: ops.Heads(v.data_ptr(), v.stride(0), v.stride(1))  # noqa: E731
    ops.rotary(gpu, t, ops.RotaryArgs(dtype=hip.F32, rows=50, q_heads=2, head_dim=16, positions=positions.data_ptr(), q_in=view(x), q_out=view(y)))
    rotary_check(y, x, positions, t, 0, "q")


# ---------------------------------------------------------------------------
# attention over packed documents
# ---------------------------------------------------------------------------

SELF = lambda *n: [(x, x) for x in n]  # noqa: E731

CASES = [
    # lens, q_heads, kv_heads, d, options
    (SELF(1), 1, 1, 8, {}),
    (SELF(5, 1, 130), 2, 2, 64, dict(mask="causal", gap=3)),
    (SELF(257, 64, 0, 31), 6, 2, 64, dict(mask="none", layout="qkv", gap=2)),
    (SELF(300), 4, 1, 128, dict(mask="causal", cap=15.0, layout="qkv")),
    (SELF(90, 129, 7), 3, 3, 40, dict(mask="prefix", bias=0.3, layout="heads", gap=1)),
    (SELF(200, 77), 4, 2, 72, dict(mask="none", bias=0.05, axes=2, cap=30.0)),
    (SELF(65, 63), 2, 1, 16, dict(mask="causal", bias=0.2, axes=3, layout="qkv")),
    (SELF(128), 1, 1, 120, dict(mask="prefix", prefix=[128], bias=0.1, axes=1)),
    ([(1, 300), (1, 1), (1, 0), (1, 64)], 8, 2, 64, dict(mask="causal", cap=20.0)),
    ([(3, 500), (0, 40), (9, 33)], 5, 1, 104, dict(mask="causal", bias=0.1, gap=4)),
    # more queries than keys: the first rows of a causal document see nothing
    ([(40, 9), (70, 64), (5, 0)], 2, 2, 32, dict(mask="causal", gap=1)),
    ([(40, 9), (66, 20)], 4, 2, 56, dict(mask="prefix", prefix=[4, 0], bias=0.2)),
    ([(33, 700)], 3, 1, 128, dict(mask="none", cap=5.0)),
    ([(150, 1000), (20, 260)], 4, 4, 64, dict(mask="prefix", prefix=[900, -3], layout="heads")),
    (SELF(700), 2, 1, 24, dict(mask="causal", spread=4.0)),
    (SELF(*([3] * 40)), 2, 2, 48, dict(mask="causal", layout="qkv")),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", range(len(CASES)))
def test_packed_attention_and_its_gradients(gpu, dtype, case):
    lens, q_heads, kv_heads, d, options = CASES[case]
    t = Packed(lens, dtype, q_heads, kv_heads, d, seed=case + 1, **options)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    t.check(["out", "lse"], False)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v", "d_slopes"], True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lens,q_heads,kv_heads,d,max_keys", [
    ([(1, 5000)], 4, 1, 128, 0), ([(1, 3000), (1, 1), (1, 0), (1, 2047)], 8, 8, 64, 3000), ([(1, 9000), (1, 10)], 6, 2, 80, 100),
    ([(4, 4097)], 12, 1, 64, 0), ([(1, 2048)] * 3, 40, 8, 128, 2048),
])
@pytest.mark.parametrize("bias", [None, 0.01])
def test_single_tokens_over_a_cache(gpu, dtype, lens, q_heads, kv_heads, d, max_keys, bias):
    t = Packed(lens, dtype, q_heads, kv_heads, d, mask="causal", cap=25.0, bias=bias, seed=3)
    ops.attention(gpu, t.args(gpu, False, max_keys))
    t.check(["out", "lse"], False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_documents_that_share_a_cache(gpu, dtype):
    """k_begin and k_end as arrays of their own: slots in another order, one
    prefix read by two documents."""
    t = Packed([(2, 64), (3, 64), (1, 200)], dtype, 4, 2, 64, mask="causal")
    w = Packed([(2, 64), (3, 64), (1, 200)], dtype, 4, 2, 64, mask="causal")
    w.k[64:128], w.v[64:128] = w.k[:64].clone(), w.v[:64].clone()
    begin = torch.tensor([0, 0, 128], device="cuda", dtype=torch.int32)
    end = begin + torch.tensor([64, 64, 200], device="cuda", dtype=torch.int32)
    a = t.args(gpu, False)
    a.k_begin, a.k_end = begin.data_ptr(), end.data_ptr()
    ops.attention(gpu, a)
    want = w.reference(False)
    assert_within(t.out, *want["out"], "out")
    assert_within(t.lse, *want["lse"], "lse")


def test_one_document_without_offsets(gpu):
    t = Packed(SELF(100), "f16", 2, 2, 64, mask="causal", bias=0.1)
    a = t.args(gpu, True)
    a.q_offsets = a.k_begin = a.k_end = None
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v", "d_slopes"], True)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_what_a_hidden_place_holds_does_not_count(gpu, dtype):
    """NaN and infinities in keys and values that the causal mask hides from a
    row, and the type's lowest value in scores, leave the rows before them
    alone."""
    t = Packed(SELF(150), dtype, 2, 1, 64, mask="causal")
    w = Packed(SELF(150), dtype, 2, 1, 64, mask="causal")
    want = w.reference(False)
    t.k[100], t.v[100] = math.nan, math.inf
    t.k[131], t.v[140] = -math.inf, math.nan
    ops.attention(gpu, t.args(gpu, False))
    assert_within(t.out[:100], want["out"][0][:100], want["out"][1][:100], "out")
    assert_within(t.lse[:, :100], want["lse"][0][:, :100], want["lse"][1][:, :100], "lse")
    assert torch.isnan(t.out[100:].float()).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_scores_far_apart_and_values_that_are_infinite(gpu, dtype):
    """A score that leaves the others no weight, and an infinite value that a
    row sees."""
    t = Packed(SELF(80), dtype, 1, 1, 16, scale=1.0)
    t.k[5] = 0.0
    t.q[:] = 0.0
    t.q[:, :, 0] = 100.0
    t.k[:, :, 0] = -100.0
    t.k[5, :, 0] = 100.0
    ops.attention(gpu, t.args(gpu, False))
    assert torch.equal(t.out[:, 0], t.v[5, 0].expand(80, 16))
    assert torch.all(t.lse == 10000.0)
    s = Packed(SELF(80), dtype, 1, 1, 16)
    s.v[7, 0, 3] = math.inf
    ops.attention(gpu, s.args(gpu, False))
    assert torch.all(s.out[:, 0, 3] == math.inf) and torch.isfinite(s.out[:, 0, :3].float()).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_small_gradients_keep_their_digits(gpu, dtype):
    """Unscaled gradients of a long row in f16: probabilities times gradients
    far below the type's smallest number, whose sums are not."""
    t = Packed(SELF(300), dtype, 2, 1, 64, mask="causal")
    size = 2.0**-13
    t.d_out *= size
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["d_q", "d_k", "d_v"], True)


def test_wrong_offsets_stay_inside_the_tensors(gpu):
    """Offsets beyond the tensors, falling and negative, are clamped: any
    result, no access outside (the rows around the tensors keep theirs)."""
    for off in ([0, 50, 20, 1000], [-7, 2**31 - 1, -2**31, 64], [60, 60, 10, 0]):
        t = Packed(SELF(20, 20, 24), "bf16", 2, 2, 64, mask="prefix", bias=0.1)
        t.q_off.copy_(torch.tensor(off))
        t.k_off.copy_(torch.tensor(off[::-1]))
        t.prefix.copy_(torch.tensor([2**31 - 1, -2**31, 5]))
        a = t.args(gpu, True)
        ops.attention(gpu, a)
        ops.attention_backward(gpu, a, t.grads())
    torch.cuda.synchronize()


def test_a_cache_beyond_32_bits(gpu):
    """Rows whose elements lie past 2^32 of the tensor's first."""
    rows, heads, d = 2**22 + 4096, 8, 128  # 2^32 elements and more, 8.6 GB a tensor
    k, v = (torch.empty(rows, heads, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    t = Packed([(2, 700)], "bf16", 16, 8, 128, mask="causal")
    first = rows - 700
    k[first:], v[first:] = t.k, t.v
    begin = torch.tensor([first], device="cuda", dtype=torch.int32)
    end = begin + 700
    a = t.args(gpu, False)
    a.k_rows, a.max_keys = rows, 700
    a.k_begin, a.k_end = begin.data_ptr(), end.data_ptr()
    a.k, a.v = (ops.Heads(x.data_ptr(), x.stride(0), x.stride(1)) for x in (k, v))
    n = ops.attention_workspace(gpu, a)
    workspace = torch.empty(n + 16, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), n
    ops.attention(gpu, a)
    t.check(["out", "lse"], False)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_repeats_bit_for_bit(gpu, dtype):
    t = Packed(SELF(400, 333), dtype, 4, 2, 64, mask="causal", bias=0.1, cap=20.0)
    a = t.args(gpu, True)
    seen = None
    for _ in range(3):
        ops.attention(gpu, a)
        ops.attention_backward(gpu, a, t.grads())
        now = [x.clone() for x in (t.out, t.lse, t.d_q, t.d_k, t.d_v, t.d_slopes)]
        assert seen is None or all(torch.equal(x, y) for x, y in zip(seen, now))
        seen = now


def test_gradients_against_differences(gpu):
    """The f32 gradients along random directions against central differences
    of the f32 forward."""
    t = Packed(SELF(40, 21), "f32", 4, 2, 32, mask="causal", cap=6.0, bias=0.2)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    g = torch.Generator(device="cuda").manual_seed(5)
    for name in ("q", "k", "v", "slopes"):
        leaf, grad = getattr(t, name), getattr(t, "d_" + name).double()
        kept = leaf.clone()
        way = torch.randn(leaf.shape, generator=g, device="cuda")
        h = 2.0**-6
        values = []
        for sign in (1, -1):
            leaf.copy_(kept + sign * h * way)
            ops.attention(gpu, a)
            values.append((t.out.double() * t.d_out.double()).sum())
        leaf.copy_(kept)
        along = (grad * way.double()).sum()
        slope = (values[0] - values[1]) / (2 * h)
        # the third derivative's h^2 / 6, of functions whose derivatives along a direction of
        # size sqrt(n) grow by a few units a step: 2^-12 / 6 of some hundreds
        size = (grad.abs() * way.double().abs()).sum()
        assert float((along - slope).abs()) <= 0.02 * float(size), name


# ---------------------------------------------------------------------------
# streams, graphs, and the operators together
# ---------------------------------------------------------------------------


def test_a_context_over_another_stream(gpu):
    side = torch.cuda.Stream()
    ctx = hip.Context(0, stream=side.cuda_stream)
    assert ctx._lib.bl_ctx_stream(ctx.handle) == side.cuda_stream
    t = Packed(SELF(200), "bf16", 2, 2, 64, mask="causal")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention(ctx, t.args(ctx, False))
    torch.cuda.current_stream().wait_stream(side)
    t.check(["out", "lse"], False)
    ctx.close()
    with torch.cuda.stream(side):  # the stream outlives the context
        x = torch.ones(4, device="cuda") * 2
    side.synchronize()
    assert float(x.sum()) == 8.0


def test_kernels_over_the_hosts_stream(gpu):
    """A program's kernels on a context over the host's stream, launched one
    by one, give what a context of its own gives."""
    import numpy as np

    from beatlm_amd import ir

    outs = []
    for ctx in (gpu, hip.Context(0)):
        g = ir.Graph()
        g.tensor(0, ir.INPUT, 33 * 64)
        g.tensor(1, ir.WEIGHT, 64)
        g.tensor(2, ir.WEIGHT, 64)
        g.tensor(3, ir.OUTPUT, 33 * 64)
        g.push(ir.op(ir.OP_LAYER_NORM, [0, 1, 2], [33, 64], 1e-6), 3)
        prep = ir.prepare(ctx, g)
        rng = np.random.default_rng(0)
        for tid, n in ((0, 33 * 64), (1, 64), (2, 64)):
            prep.write(tid, rng.standard_normal(n).astype(np.float32))
        prep.run()
        ctx.synchronize()
        outs.append(prep.read(3))
        prep.close()
    assert np.array_equal(*outs)


def test_captured_and_replayed(gpu):
    """Forward and backward in one graph, replayed with other inputs and other
    offsets, between eager work."""
    t = Packed(SELF(150, 90), "bf16", 4, 2, 64, mask="causal", bias=0.1)
    n = Norm(300, 384, "bf16")
    stream = torch.cuda.Stream()
    ctx = hip.Context(0, stream=stream.cuda_stream)
    a, g, na = t.args(ctx, True), t.grads(), n.args()
    ng = n.grads(ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.layer_norm(ctx, na)
        ops.attention(ctx, a)
        ops.attention_backward(ctx, a, g)
        ops.layer_norm_backward(ctx, na, ng)
    for step, lens in enumerate([SELF(150, 90), SELF(10, 230), SELF(240, 0), SELF(77, 100)]):
        w = Packed(lens, "bf16", 4, 2, 64, mask="causal", bias=0.1, seed=20 + step)
        for name in ("q", "k", "v", "d_out"):
            getattr(t, name).zero_()
            getattr(t, name)[: getattr(w, name).shape[0]] = getattr(w, name)
        t.slopes.copy_(w.slopes)
        t.q_off.copy_(w.q_off)
        t.k_off.copy_(w.k_off)
        n.x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = w.reference(True)
        for name in ("out", "d_q", "d_k", "d_v"):
            rows = want[name][0].shape[0]
            assert_within(getattr(t, name)[:rows], *want[name], f"replay {step}: {name}")
        assert_within(t.d_slopes, *want["d_slopes"], f"replay {step}: d_slopes")
        n.check()
    ctx.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_sublayer_s_training_step(gpu, dtype):
    """LayerNorm, the projection (torch's), rotary positions in place and
    attention over packed images, and back: every gradient against the whole
    chain's in 64 bits."""
    torch_dtype, code = DTYPES[dtype]
    images, heads, kv, d, width = [(5, 7), (3, 3), (8, 6)], 4, 2, 32, 96
    rows = sum(h * w for h, w in images)
    g = torch.Generator(device="cuda").manual_seed(9)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch_dtype)  # noqa: E731
    x, gamma, beta, d_out = make(rows, width), make(width) * 0.2 + 1, make(width) * 0.2, make(rows, heads, d)
    weight = make(width, (heads + 2 * kv) * d) * 0.1
    positions = torch.cat([torch.stack([torch.arange(h * w) // w, torch.arange(h * w) % w], 1) for h, w in images]).to("cuda", torch.int32).contiguous()
    offsets = torch.tensor([0] + [h * w for h, w in images], device="cuda").cumsum(0).to(torch.int32)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.02], device="cuda")
    view = lambda t: ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
    empty = lambda *s: torch.empty(*s, device="cuda", dtype=torch_dtype)  # noqa: E731
    f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731

    normed, mean, rstd = empty(rows, width), f32(rows), f32(rows)
    na = ops.LayerNormArgs(dtype=code, rows=rows, cols=width, epsilon=1e-6, x_stride=width, y_stride=width, x=x.data_ptr(), gamma=gamma.data_ptr(),
                           beta=beta.data_ptr(), y=normed.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr())
    ops.layer_norm(gpu, na)
    qkv = (normed.float() @ weight.float()).to(torch_dtype).view(rows, heads + 2 * kv, d)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    table = ops.rotary_table([8, 8], 100.0, per_axis=True)
    turn = dict(dtype=code, rows=rows, q_heads=heads, k_heads=kv, head_dim=d, positions=positions.data_ptr())
    ops.rotary(gpu, table, ops.RotaryArgs(q_in=view(q), q_out=view(q), k_in=view(k), k_out=view(k), **turn))
    out, lse = empty(rows, heads, d), f32(heads, rows)
    a = ops.AttentionArgs(dtype=code, q_heads=heads, kv_heads=kv, head_dim=d, q_rows=rows, k_rows=rows, documents=len(images), axes=2, scale=d**-0.5,
                          q_offsets=offsets.data_ptr(), k_begin=offsets.data_ptr(), k_end=offsets.data_ptr() + 4, slopes=slopes.data_ptr(),
                          q_positions=positions.data_ptr(), k_positions=positions.data_ptr(), q=view(q), k=view(k), v=view(v), out=view(out),
                          lse=lse.data_ptr())
    n = ops.attention_workspace(gpu, a, True)
    workspace = torch.empty(n + 16, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), n
    ops.attention(gpu, a)
    d_qkv, d_slopes = torch.zeros_like(qkv), f32(heads)
    dq, dk, dv = d_qkv[:, :heads], d_qkv[:, heads:heads + kv], d_qkv[:, heads + kv:]
    ops.attention_backward(gpu, a, ops.AttentionGrads(d_out=view(d_out), d_q=view(dq), d_k=view(dk), d_v=view(dv), d_slopes=d_slopes.data_ptr()))
    ops.rotary(gpu, table, ops.RotaryArgs(q_in=view(dq), q_out=view(dq), k_in=view(dk), k_out=view(dk), inverse=1, **turn))
    d_normed = (d_qkv.view(rows, -1).float() @ weight.float().T.contiguous()).to(torch_dtype)
    dx, d_gamma, d_beta = empty(rows, width), f32(width), f32(width)
    m = ops.layer_norm_backward_workspace(gpu, na)
    scratch = torch.empty(m + 16, device="cuda", dtype=torch.uint8)
    ops.layer_norm_backward(gpu, na, ops.LayerNormGrads(dy=d_normed.data_ptr(), dy_stride=width, dx=dx.data_ptr(), dx_stride=width,
                                                        d_gamma=d_gamma.data_ptr(), d_beta=d_beta.data_ptr(), workspace=scratch.data_ptr(), workspace_bytes=m))

    lx, lg, lb, lw, ls = (t.double().cpu().requires_grad_() for t in (x, gamma, beta, weight, slopes))
    mu = lx.mean(1, keepdim=True)
    y = (lx - mu) * (((lx - mu) ** 2).mean(1, keepdim=True) + 1e-6).rsqrt() * lg + lb
    z = (y @ lw).view(rows, heads + 2 * kv, d)
    turns = torch.tensor(list(table.turns[:16]), dtype=torch.float64) * 2 * math.pi
    phi = (positions.cpu().double()[:, list(table.axis[:16])] * turns)[:, None]
    a0, b0 = z[:, :heads + kv, :16], z[:, :heads + kv, 16:]
    qk = torch.cat([a0 * phi.cos() - b0 * phi.sin(), a0 * phi.sin() + b0 * phi.cos()], -1)
    doc = torch.repeat_interleave(torch.arange(len(images)), torch.tensor([h * w for h, w in images]))
    far = (positions.cpu().double()[:, None] - positions.cpu().double()[None]).abs().sum(-1)
    o = []
    for h in range(heads):
        s = qk[:, h] @ qk[:, heads + h // 2].T * d**-0.5 - ls[h] * far
        s = s.masked_fill(doc[:, None] != doc[None], -math.inf)
        o.append(s.softmax(1) @ z[:, heads + kv + h // 2])
    o = torch.stack(o, 1)
    want = torch.autograd.grad(o, (lx, lg, lb, ls), d_out.double().cpu())
    # Chained roundings to the type: four on the way there, four on the way back; in the 2-norm each
    # adds at most half a step of what passes through (f32: its sums of up to 200 products instead).
    most = 16 * half_step(torch_dtype) if torch_dtype != torch.float32 else 400 * F32
    for name, got, w in (("out", out, o.detach()), ("dx", dx, want[0]), ("d_gamma", d_gamma, want[1]), ("d_beta", d_beta, want[2]), ("d_slopes", d_slopes, want[3])):
        off = float((got.double().cpu() - w).norm() / w.norm())
        assert off <= most, (name, off, most)


# ---------------------------------------------------------------------------
# where it can go wrong
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_a_single_key_takes_all_the_weight(gpu, dtype, d, mask):
    """One visible key: its value comes out as it is, and no gradient reaches
    the scores, exactly."""
    t = Packed([(1, 1)] * 70 + [(7, 1) if mask == "none" else (1, 1)], dtype, 4, 2, d, mask=mask, cap=9.0, bias=0.2)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_v"], True)
    assert torch.equal(t.out[:70], t.v[:70].repeat_interleave(2, 1))
    for grad in (t.d_q, t.d_k, t.d_slopes):
        assert torch.all(grad == 0.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("mask,prefix", [("causal", None), ("prefix", [1, 0])])
def test_rows_of_one_key_or_none_among_others(gpu, dtype, mask, prefix):
    """More queries than keys: rows that see nothing, with NaN in them, and
    rows that see one key, before rows that see more."""
    lens = [(45, 9), (70, 66)]
    t, w = (Packed(lens, dtype, 2, 1, 64, mask=mask, prefix=prefix) for _ in range(2))
    dead = [i for i in range(36)] if prefix is None else []
    dead += [45 + i for i in range(4)]
    one = [36] if prefix is None else list(range(37))
    one += [45 + 4]
    t.q[dead], t.d_out[dead] = math.nan, math.nan
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    want = w.reference(True)
    for name in ("out", "lse", "d_q", "d_k", "d_v"):
        assert_within(getattr(t, name), *want[name], name)
    assert torch.all(t.out[dead] == 0.0) and torch.all(t.lse[:, dead] == -math.inf)
    assert torch.all(t.d_q[dead + one] == 0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("documents,heads", [(200, 2), (4300, 1)])
def test_many_documents(gpu, dtype, documents, heads):
    t = Packed([(i % 4, i % 4) for i in range(documents)], dtype, heads, 1, 16, mask="causal")
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v"], True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("options", [dict(), dict(cap=7.0), dict(bias=0.1)])
def test_scales_below_and_at_zero(gpu, dtype, scale, options):
    t = Packed(SELF(90, 33), dtype, 2, 1, 64, mask="causal", scale=scale, **options)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v", "d_slopes"], True)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("axes", [0, 1, 2, 3])
@pytest.mark.parametrize("d", [40, 128])
def test_few_tokens_with_a_bias_and_hidden_places(gpu, dtype, axes, d):
    """A decoding step's chunk, whose last key its earlier rows do not see,
    whatever that holds."""
    lens = [(4, 500), (1, 77), (3, 130), (2, 3)]
    t, w = (Packed(lens, dtype, 6, 3, d, mask="causal", bias=0.1, axes=axes, gap=2) for _ in range(2))
    last = [2 + 499, 2 + 500 + 77 + 129, 2 + 500 + 77 + 130 + 2]
    t.k[last], t.v[last] = math.nan, math.inf
    ops.attention(gpu, t.args(gpu, False, 500))
    want = w.reference(False)
    clean = [2, 3, 4, 6, 7, 8, 10]  # rows 2 to 5, 6, 7 to 9 and 10 to 11, without each chunk's last
    assert_within(t.out[clean], want["out"][0][clean], want["out"][1][clean], "out")
    assert_within(t.lse[:, clean], want["lse"][0][:, clean], want["lse"][1][:, clean], "lse")
    assert torch.all(t.out[:2] == 7.0) and torch.all(t.out[-2:] == 7.0)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_tensors_without_rows(gpu, dtype):
    t = Packed([(5, 0), (3, 0)], dtype, 2, 1, 64)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    assert torch.all(t.out == 0.0) and torch.all(t.lse == -math.inf) and torch.all(t.d_q == 0.0)
    t = Packed([(0, 5), (0, 130)], dtype, 2, 1, 64, mask="causal", bias=0.1)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    assert torch.all(t.d_k == 0.0) and torch.all(t.d_v == 0.0) and torch.all(t.d_slopes == 0.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("lens,d", [([(1, 3000)], 128), ([(70, 900)], 64), ([(700, 700)], 128)])
def test_a_workspace_is_as_large_as_it_says(gpu, dtype, lens, d):
    t = Packed(lens, dtype, 4, 2, d, mask="causal", bias=0.1)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    assert torch.all(t.workspace[-16:] == 0xFF)
    n = Norm(700, 200, dtype)
    ops.layer_norm(gpu, n.args())
    ops.layer_norm_backward(gpu, n.args(), n.grads(gpu))
    assert torch.all(n.workspace[-16:] == 0xFF)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_key_head_that_is_broadcast(gpu, dtype):
    """Two key heads that are one tensor's, read through a head stride of
    zero: each keeps the gradients of its own queries."""
    t, w = (Packed(SELF(100, 57), dtype, 4, 2, 64, mask="causal") for _ in range(2))
    for x in (w.k, w.v):
        x[:, 1] = x[:, 0]
    a = t.args(gpu, True)
    a.k.head_stride = a.v.head_stride = 0
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    want = w.reference(True)
    for name in ("out", "lse", "d_q", "d_k", "d_v"):
        assert_within(getattr(t, name), *want[name], name)


def test_two_streams_at_once(gpu):
    """Calls that overlap in time, a workspace each, give the bits of calls in
    turn."""
    problems = [Packed(SELF(300, 200), "bf16", 4, 2, 128, mask="causal", cap=20.0, seed=s) for s in (1, 2)]
    ready = [(t, t.args(gpu, True), t.grads()) for t in problems]
    want = []
    for t, a, g in ready:
        ops.attention(gpu, a)
        ops.attention_backward(gpu, a, g)
        want.append([x.clone() for x in (t.out, t.lse, t.d_q, t.d_k, t.d_v)])
        for x in (t.out, t.lse, t.d_q, t.d_k, t.d_v):
            x.zero_()
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [hip.Context(0, stream=s.cuda_stream) for s in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for ctx, (t, a, g) in zip(contexts, ready):
            ops.attention(ctx, a)
            ops.attention_backward(ctx, a, g)
    torch.cuda.synchronize()
    for (t, _, _), kept in zip(ready, want):
        assert all(torch.equal(x, y) for x, y in zip((t.out, t.lse, t.d_q, t.d_k, t.d_v), kept))
    for ctx in contexts:
        ctx.close()


def test_rotary_of_more_rows_than_a_grid_has_threads(gpu):
    """One pair of a head of 256, a workgroup a row: 2^23 of them and some."""
    rows = 2**23 + 7
    x = torch.ones(rows, 1, 256, device="cuda", dtype=torch.float16)
    x[:, 0, 1] = 0.0
    positions = (torch.arange(rows, device="cuda", dtype=torch.int32) % 1000).contiguous()
    view = ops.Heads(x.data_ptr(), 256, 256)
    ops.rotary(gpu, ops.rotary_table([1], 10.0), ops.RotaryArgs(dtype=hip.F16, rows=rows, q_heads=1, head_dim=256, positions=positions.data_ptr(), q_in=view, q_out=view))
    phi = positions.double()
    # a sine of f32 in 64-bit reduced angles, rounded once
    for c, want in ((0, phi.cos()), (1, phi.sin())):
        assert_within(x[:, 0, c], want, half_step(torch.float16) * want.abs() + 16 * F32 + 2.0**-25, f"channel {c}")
    assert torch.all(x[-9:, 0, 2:] == 1.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("d,keys", [(16, 60), (128, 60), (64, 1000)])
def test_the_slopes_gradient_does_not_see_the_statistics_rounding(gpu, dtype, d, keys):
    """Keys of one value leave the scores without gradient, whatever P is. lse
    is about 2000 here, so rounding it to f32 scales a row's P by up to 2^-13."""
    t = Packed([(1, keys)], dtype, 8, 2, d, bias=0.02, scale=1.0)
    t.q[..., 0], t.k[..., 0] = 45.0, 45.0
    t.v[:] = t.v[:1].clone()
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    far = (keys - 1 - torch.arange(keys, device="cuda")).double()
    for h in range(8):
        q, k = t.q[0, h].double(), t.k[:, h // 4].double()
        p = (k @ q - float(t.slopes[h]) * far).softmax(0)
        dp = float((t.d_out[0, h].double().abs() * t.v[0, h // 4].double().abs()).sum())
        # three sums of `keys` terms in f32, and a few products
        most = (3 * keys + 16) * F32 * dp * float((p * far).sum())
        assert abs(float(t.d_slopes[h])) <= most, (h, float(t.d_slopes[h]), most)
