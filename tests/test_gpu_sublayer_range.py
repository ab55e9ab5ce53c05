"""The packed sublayer's operators where numbers come near the ends of their
types, against their formulas in 64 bits."""

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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [16, 64, 72, 128])
@pytest.mark.parametrize("queries", [1, 40])
def test_scores_gradients_beyond_the_type_s_range(gpu, dtype, d, queries):
    """Two keys of equal weight whose values are far apart in every channel,
    under gradients of 1: a score's gradient is 2^17, beyond f16, and d_q, a few
    thousand to 2^15, is not."""
    t = Packed([(queries, 2)] * 2, dtype, 2, 1, d, seed=d)
    t.q.zero_()
    t.q[..., 0] = 2.0**-6
    t.k[:] = torch.rand(4, 1, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) - 0.5
    t.k[..., 0] = 0.0  # scores of 0
    t.v[0::2], t.v[1::2] = 2.0**18 / d, -(2.0**18) / d
    t.d_out.fill_(1.0)
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    assert float(t.d_q.float().abs().max()) > 1000.0
    t.check(["out", "lse", "d_q", "d_k", "d_v"], True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", ["none", "causal"])
def test_gradients_under_large_values(gpu, dtype, d, mask):
    """Values in the ten thousands over few keys, and over many in documents of
    one batch, beside a document of ordinary ones."""
    t = Packed([(3, 2), (5, 5), (40, 40), (70, 300), (20, 20)], dtype, 4, 2, d, mask=mask)
    t.q *= 0.25
    t.k *= 0.25
    t.v[:-20] *= 8192.0
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    t.check(["out", "lse", "d_q", "d_k", "d_v"], True)


# Flat rows over so many keys that each probability is 100.5 of f16's smallest steps
LONG = 166937
# what f32 may put on a sum over them: at most 1024 splits, joined in turn, of at most 192 keys
SUMS = F32 * (1024 + 192 + 64)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_long_flat_rows_keep_their_digits(gpu, dtype, d):
    t = Packed([(3, LONG)], dtype, 1, 1, d)
    t.q.zero_()
    t.q[..., 0] = 1.0
    t.k[..., 0] = 0.0
    t.d_out *= 1000.0
    a = t.args(gpu, True)
    ops.attention(gpu, a)
    ops.attention_backward(gpu, a, t.grads())
    u, p, scale = half_step(t.torch_dtype), 1.0 / LONG, d**-0.5
    q, k, v, g = (x[:, 0].double() for x in (t.q, t.k, t.v, t.d_out))
    # P once rounded for the products, the output once
    want = p * g.sum(0).expand(LONG, d)
    assert_within(t.d_v[:, 0], want, u * want.abs() + (u + SUMS) * p * g.abs().sum(0), "d_v")
    dp, size = g @ v.T, g.abs() @ v.abs().T
    ds = p * (dp - dp.mean(1, keepdim=True))
    # dS is off by its own rounding and by its sums', and by f16's smallest step, 2^-25, of 2^-10 of
    # twice a bound of |dP|
    bound = 2 * g.norm(dim=1, keepdim=True) * v.norm(dim=1).max()
    off = u * ds.abs() + p * SUMS * (size + size.mean(1, keepdim=True)) + (2.0**-35 * bound if dtype == "f16" else 0.0)
    want = scale * ds.T @ q
    assert_within(t.d_k[:, 0], want, u * want.abs() + scale * off.T @ q.abs() + 2.0**-25, "d_k")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_long_tail_of_small_probabilities_keeps_its_digits(gpu, dtype):
    """One key ahead of all others, which have half the weight together: each is
    101.48 of f16's smallest steps beside the first. 256 heads on one key head's
    tensors, so that no split takes the tail apart."""
    heads, d = 256, 64
    t = Packed([(1, LONG)], dtype, heads, 1, d, scale=1.0)
    t.q.zero_()
    t.q[..., 0] = 1.0
    t.k.zero_()
    t.k[0, 0, 0] = 12.015625
    t.v[:], t.v[0] = 1.0, 0.0
    a = t.args(gpu, False)
    a.kv_heads = heads
    a.k.head_stride = a.v.head_stride = 0
    n = ops.attention_workspace(gpu, a)
    workspace = torch.empty(n + 16, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), n
    ops.attention(gpu, a)
    u = half_step(t.torch_dtype)
    first = float(t.k[0, 0, 0].double())
    tail = (LONG - 1) * torch.tensor(-first, dtype=torch.float64).exp().item()
    want = torch.full_like(t.out, tail / (1 + tail), dtype=torch.float64)
    # P once rounded, the output once; unsplit sums of equal terms in f32, a lane's 32 of 64 keys a tile
    assert_within(t.out, want, want * (2 * u + F32 * (LONG / 2 + 64)), "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [5, 200, 1003, 4099])
def test_layer_norm_s_gradients_of_flat_rows_of_large_values(gpu, dtype, cols):
    """x is its mean everywhere, so n is 0, and mean times rstd is beyond f32."""
    torch_dtype, code = DTYPES[dtype]
    rows, epsilon = 3, 1e-6
    g = torch.Generator(device="cuda").manual_seed(cols)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch_dtype)  # noqa: E731
    x = torch.full((rows, cols), 2.0**121, device="cuda", dtype=torch_dtype)
    dy, gamma, dx = make(rows, cols), make(cols), torch.empty_like(x)
    mean, rstd = torch.full((rows,), 2.0**121, device="cuda"), torch.full((rows,), epsilon**-0.5, device="cuda")
    d_gamma, d_beta = (torch.empty(cols, device="cuda") for _ in range(2))
    a = ops.LayerNormArgs(dtype=code, rows=rows, cols=cols, epsilon=epsilon, x_stride=cols, x=x.data_ptr(), gamma=gamma.data_ptr(),
                          mean=mean.data_ptr(), rstd=rstd.data_ptr())
    n = ops.layer_norm_backward_workspace(gpu, a)
    workspace = torch.empty(n, device="cuda", dtype=torch.uint8)
    ops.layer_norm_backward(gpu, a, ops.LayerNormGrads(dy=dy.data_ptr(), dy_stride=cols, dx=dx.data_ptr(), dx_stride=cols, d_gamma=d_gamma.data_ptr(),
                                                       d_beta=d_beta.data_ptr(), workspace=workspace.data_ptr(), workspace_bytes=n))
    scaled, r = dy.double() * gamma.double(), rstd.double()[:, None]
    want = r * (scaled - scaled.mean(1, keepdim=True))
    # a sum of 16 values a thread and at most 22 additions of those, one product and one difference each
    off = r * F32 * (40 * scaled.abs().mean(1, keepdim=True) + 4 * scaled.abs())
    assert_within(dx, want, half_step(torch_dtype) * want.abs() + off, "dx")
    assert torch.all(d_gamma == 0.0)
    assert_within(d_beta, dy.double().sum(0), F32 * (rows + 8) * dy.double().abs().sum(0), "d_beta")


@pytest.mark.parametrize("axes", [0, 1, 2, 3])
def test_few_tokens_over_many_blocks_of_keys(gpu, axes):
    """f32, so many documents that no split cuts the keys short: a wave goes
    through dozens of blocks with the next one's loads under way."""
    t = Packed([(1 + i % 3, 1500 + 37 * i) for i in range(34)], "f32", 8, 8, 64, mask="causal", bias=0.02, axes=axes, gap=1)
    a = t.args(gpu, False)
    ops.attention(gpu, a)
    t.check(["out", "lse"], False)
    first = t.out.clone(), t.lse.clone()
    for _ in range(5):
        ops.attention(gpu, a)
        assert torch.equal(t.out, first[0]) and torch.equal(t.lse, first[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keys", [1, 300])
def test_statistics_near_zero_keep_their_digits(gpu, dtype, keys):
    """Scores and lse of 2^-12 and less: lse is the score itself over one key, and
    keys whose number the bias of the first cancels leave nothing else."""
    t = Packed([(1, keys)] * 20, dtype, 2, 1, 16, scale=1.0)
    t.q.zero_()
    t.k.zero_()
    t.q[..., 0] = 2.0**-6
    t.k[:, :, 0] = (torch.rand(t.k_rows, 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 2.0**-6).to(t.torch_dtype)
    if keys > 1:  # all but the first of a document far below it
        t.q[..., 1] = 64.0
        t.k[:, :, 1] = -8.0
        t.k[0::keys, :, 1] = 0.0
    ops.attention(gpu, t.args(gpu, False))
    first = t.k[0::keys, 0].double()
    want = (t.q[..., 0].double() * first[:, None, 0]).T  # one product, exact in f32
    # into base two, and out of it again: a few roundings of it, and the hardware's log2 of a sum of 1
    assert_within(t.lse, want, 6 * F32 * want.abs(), "lse")
