"""Norms of heads with their rotary positions, and the gradients
(include/beatlm_cache.h), against their formulas in 64 bits."""

import math

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import EPSILON, NORMS, SENTINEL, angles, at, heads, ints, normed, spread, tiny, turn_tolerance, turned
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


class Heads:
    """q and k as views with gaps, in either order of rows and heads."""

    def __init__(self, dtype, rows, q_heads, k_heads, d, sections, norm="rms", neighbours=False, layout="qkv", start=0, seed=1, weights=True, offset=0.0):
        self.torch_dtype, self.dtype = DTYPES[dtype]
        self.rows, self.q_heads, self.k_heads, self.d, self.norm, self.neighbours = rows, q_heads, k_heads, d, norm, neighbours
        self.table = ops.rotary_table(sections, 10000.0, neighbours=neighbours) if sections else None
        g = torch.Generator(device="cuda").manual_seed(seed)

        def tensor(n, fill=SENTINEL, pad=8):
            if layout == "heads":
                return torch.full((n, rows, d), fill, device="cuda", dtype=self.torch_dtype).permute(1, 0, 2)
            return torch.full((rows, n + 2, d + pad), fill, device="cuda", dtype=self.torch_dtype)[:, 1:1 + n, :d]

        def random(n, size=1.0, by=0.0):
            t = tensor(n, math.nan, 1 if layout == "odd" else 8)
            t.copy_((torch.randn(rows, n, d, generator=g, device="cuda") * size + by).to(self.torch_dtype))
            return t

        self.x = [random(q_heads, 1.3, offset), random(k_heads, 0.4, offset)]
        self.dy = [random(q_heads), random(k_heads)]
        self.y, self.dx = ([tensor(q_heads), tensor(k_heads)] for _ in range(2))
        make = lambda: (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(self.torch_dtype) if weights else None  # noqa: E731
        self.gamma = [make(), make()]
        self.d_gamma = [torch.full((d,), SENTINEL, device="cuda") for _ in range(2)]
        axes = len(sections) or 1
        self.positions = torch.randint(-50, 5000, (rows, axes), generator=g, device="cuda", dtype=torch.int32) + start

    def args(self):
        return ops.HeadNormArgs(dtype=self.dtype, rows=self.rows, q_heads=self.q_heads, k_heads=self.k_heads, head_dim=self.d, norm=NORMS[self.norm],
                                epsilon=EPSILON, positions=at(self.positions), q_gamma=at(self.gamma[0]), k_gamma=at(self.gamma[1]),
                                q_in=heads(self.x[0]), q_out=heads(self.y[0]), k_in=heads(self.x[1]), k_out=heads(self.y[1]))

    def grads(self, ctx):
        n = ops.head_norm_rotary_backward_workspace(ctx, self.args())
        self.workspace = torch.full((n + 512,), 0xFF, device="cuda", dtype=torch.uint8)
        return ops.HeadNormGrads(dq_out=heads(self.dy[0]), dk_out=heads(self.dy[1]), dq_in=heads(self.dx[0]), dk_in=heads(self.dx[1]),
                                 d_q_gamma=at(self.d_gamma[0]), d_k_gamma=at(self.d_gamma[1]), workspace=self.workspace.data_ptr() + 256, workspace_bytes=n)

    def check(self, backward=True):
        u, small = half_step(self.torch_dtype), tiny(self.torch_dtype)
        one = torch.ones(self.rows, 0, device="cuda", dtype=torch.float64)
        cos, sin = angles(self.table, self.positions) if self.table else (one, one)
        epsilon = torch.tensor(EPSILON, dtype=torch.float32).double().item()
        assert abs(epsilon - EPSILON) < 1e-12
        for x, dy, y, dx, gamma, d_gamma in zip(self.x, self.dy, self.y, self.dx, self.gamma, self.d_gamma):
            x, dy = x.double(), dy.double()
            gamma = gamma.double() if gamma is not None else torch.ones(self.d, device="cuda", dtype=torch.float64)
            n, n_off, rstd, rstd_off = normed(x, self.norm)
            z = n * gamma
            z_off = n_off * gamma.abs() + 2 * F32 * z.abs()
            want = turned(z, cos, sin, self.neighbours)
            assert_within(y, want, u * want.abs() + turn_tolerance(z, z_off, self.table, self.neighbours) + small, "y")
            if not backward:
                continue
            dz = turned(dy, cos, -sin, self.neighbours)
            dz_off = 8 * F32 * (spread(dy.abs(), self.table.pairs, self.neighbours) if self.table else dy.abs())
            g, g_off = dz * gamma, dz_off * gamma.abs() + F32 * (dz * gamma).abs()
            mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
            along = mean(g * n)
            along_off = mean(g_off * n.abs() + g.abs() * n_off) + 26 * F32 * mean((g * n).abs())
            centre = mean(g) if self.norm == "centred" else torch.zeros_like(along)
            centre_off = mean(g_off) + 26 * F32 * mean(g.abs()) if self.norm == "centred" else torch.zeros_like(along)
            want = rstd * (g - centre - n * along)
            size = g.abs() + centre.abs() + n.abs() * along.abs()
            off = rstd * (g_off + centre_off + n_off * along.abs() + n.abs() * along_off + 6 * F32 * size) + rstd_off * size
            assert_within(dx, want, u * want.abs() + off + small, "dx")
            if x.shape[1] == 0:  # a tensor of no heads and its weights are not touched
                assert torch.all(d_gamma == SENTINEL)
                continue
            count = x.shape[0] * x.shape[1]
            assert_within(d_gamma, (dz * n).sum((0, 1)), F32 * (count + 8) * (dz * n).abs().sum((0, 1)) + (dz.abs() * n_off + dz_off * n.abs()).sum((0, 1)) + 1e-30, "d_gamma")
        if backward:
            assert torch.all(self.workspace[:256] == 0xFF) and torch.all(self.workspace[-256:] == 0xFF)


SHAPES = [
    # rows, q_heads, k_heads, d, sections, neighbours, layout
    (1, 1, 1, 16, [8], False, "qkv"), (5, 16, 4, 128, [64], False, "qkv"), (37, 3, 1, 64, [16, 16], True, "heads"), (9, 9, 3, 80, [20], True, "qkv"),
    (2, 2, 2, 256, [128], False, "qkv"), (3, 1, 2, 256, [1], True, "odd"), (6, 4, 4, 40, [5, 4, 3], False, "qkv"), (300, 6, 2, 72, [36], False, "qkv"),
    (4, 2, 1, 8, [], False, "qkv"), (7, 3, 3, 254, [100], False, "odd"), (1025, 5, 1, 96, [24], True, "heads"), (11, 2, 2, 3, [1], False, "odd"),
    (64, 0, 3, 128, [32, 32], False, "qkv"), (64, 3, 0, 120, [60], True, "qkv"), (4500, 2, 1, 32, [16], False, "qkv"), (13, 4, 2, 1, [], False, "odd"),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("norm", ["rms", "centred"])
@pytest.mark.parametrize("shape", SHAPES)
def test_heads_and_their_gradients(gpu, dtype, norm, shape):
    rows, q_heads, k_heads, d, sections, neighbours, layout = shape
    t = Heads(dtype, rows, q_heads, k_heads, d, sections, norm, neighbours, layout)
    ops.head_norm_rotary(gpu, t.table, t.args())
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), t.grads(gpu))
    t.check()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_without_weights_and_far_positions(gpu, dtype):
    t = Heads(dtype, 33, 4, 2, 64, [32], "rms", weights=False, start=2_000_000)
    ops.head_norm_rotary(gpu, t.table, t.args())
    g = t.grads(gpu)
    g.d_k_gamma = None  # not wanted
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), g)
    assert torch.all(t.d_gamma[1] == SENTINEL)
    g.d_k_gamma = at(t.d_gamma[1])
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), g)
    t.check()


def test_a_large_offset_keeps_the_centred_variance(gpu):
    t = Heads("f32", 40, 2, 2, 128, [64], "centred", offset=300.0)
    ops.head_norm_rotary(gpu, t.table, t.args())
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), t.grads(gpu))
    t.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(gpu, dtype):
    """y over x; dx over dy, and over x."""
    make = lambda: Heads(dtype, 21, 4, 2, 96, [48], "centred")  # noqa: E731
    w = make()
    ops.head_norm_rotary(gpu, w.table, w.args())
    ops.head_norm_rotary_backward(gpu, w.table, w.args(), w.grads(gpu))
    t = make()
    a = t.args()
    a.q_out, a.k_out = a.q_in, a.k_in
    ops.head_norm_rotary(gpu, t.table, a)
    assert all(torch.equal(x, y) for x, y in zip(t.x, w.y))
    for which in ("x", "dy"):
        t = make()
        g = t.grads(gpu)
        g.dq_in, g.dk_in = (heads(v) for v in getattr(t, which))
        ops.head_norm_rotary_backward(gpu, t.table, t.args(), g)
        assert all(torch.equal(x, y) for x, y in zip(getattr(t, which), w.dx))


def test_no_rows_clear_the_weights_gradients(gpu):
    t = Heads("bf16", 1, 2, 2, 64, [32])
    a = t.args()
    a.rows = 0
    ops.head_norm_rotary(gpu, t.table, a)
    ops.head_norm_rotary_backward(gpu, t.table, a, t.grads(gpu))
    assert all(torch.all(v == 0) for v in t.d_gamma) and all(torch.all(v == SENTINEL) for v in t.y + t.dx)


def test_gradients_repeat_bit_for_bit(gpu):
    got = []
    for _ in range(3):
        t = Heads("f16", 3001, 6, 2, 64, [32])
        ops.head_norm_rotary_backward(gpu, t.table, t.args(), t.grads(gpu))
        got.append([v.clone() for v in t.dx + t.d_gamma])
    assert all(torch.equal(x, y) for other in got[1:] for x, y in zip(got[0], other))


def test_gradients_against_differences(gpu):
    """<dy, y(x + e v) - y(x - e v)> / 2e, from the 64-bit formula, is <dx, v>; the same for the weights."""
    t = Heads("f32", 6, 2, 1, 32, [12], "centred")
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), t.grads(gpu))
    cos, sin = angles(t.table, t.positions)
    g = torch.Generator(device="cuda").manual_seed(9)
    for n in range(2):
        x, dy, gamma = t.x[n].double(), t.dy[n].double(), t.gamma[n].double()
        y = lambda x, gamma: turned(normed(x, "centred")[0] * gamma, cos, sin, False)  # noqa: E731
        e = 1e-5
        for leaf, grad in (("x", t.dx[n]), ("gamma", t.d_gamma[n])):
            v = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
            up, down = (y(x + s * v, gamma) if leaf == "x" else y(x, gamma + s * v) for s in (e, -e))
            want = float((dy * (up - down)).sum() / (2 * e))
            # the difference's own error is e^2, and f32's 2^-24 of the sum's magnitude a few times over
            size = float((grad.double() * v).abs().sum())
            assert abs(float((grad.double() * v).sum()) - want) < 64 * F32 * size + 1e-7 * abs(want) + 1e-8, leaf


def test_captured_and_replayed(gpu):
    t = Heads("bf16", 50, 4, 2, 128, [64])
    stream = torch.cuda.Stream()
    ctx = hip.Context(0, stream=stream.cuda_stream)
    a, g = t.args(), t.grads(ctx)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.head_norm_rotary(ctx, t.table, a)
        ops.head_norm_rotary_backward(ctx, t.table, a, g)
    for seed in (5, 6, 7):
        fresh = Heads("bf16", 50, 4, 2, 128, [64], seed=seed)
        for mine, other in zip(t.x + t.dy + t.gamma + [t.positions], fresh.x + fresh.dy + fresh.gamma + [fresh.positions]):
            mine.copy_(other)
        for v in t.y + t.dx + t.d_gamma:
            v.fill_(SENTINEL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        t.check()
    ctx.close()
