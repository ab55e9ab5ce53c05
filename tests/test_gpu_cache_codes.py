"""4-bit groups at the ends of f16's range: up to where they stand for finite values."""

import pytest
import torch

from beatlm_amd import hip, ops
from tests.cachedata import SENTINEL, Cache, heads

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


def test_groups_up_to_65440_stand_for_finite_values(gpu):
    """A group's low and step are each rounded to f16, by up to 16 and 4: its last
    code stands for at most 65440 + 16 + 15 * 4 = 65516, under 65520, where f16
    rounds to infinity. A value is off by half a step, low's and step's roundings
    and its own in f16: (range / 15) / 2 + 16 + 15 * 4 + 16."""
    n, d = 512, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    ends = (torch.rand(n, d // 32, 2, generator=g, device="cuda") * 2 - 1) * 65440
    ends[:256, :, 1] = 65440.0
    ends[256:320, :, 0] = -65440.0
    ends[:64, :, 0] = 32768 + 32 * torch.arange(64, device="cuda")[:, None] + 16.5  # low rounds up by nearly 16
    ends[64:128, :, 0] = -65440 + 32.0 * torch.arange(64, device="cuda")[:, None]
    x = ends[..., :1] + (ends[..., 1:] - ends[..., :1]) * torch.linspace(0, 1, 32, device="cuda")
    x[..., 0], x[..., -1] = ends[..., 0], ends[..., 1]
    x = x.flatten(-2).clamp(-65440, 65440)
    cache = Cache([n], "f32", "int4", 1, d, 16, fill=False)
    k, v = x[:, None].contiguous(), -x[:, None].contiguous()
    out = [torch.full((n, 1, d), SENTINEL, device="cuda") for _ in range(2)]
    ops.cache_append(gpu, None, ops.CacheAppendArgs(dtype=hip.F32, rows=n, documents=1, q_heads=0, kv_heads=1, head_dim=d, norm=ops.HEAD_NORM_NONE,
                                                    k_in=heads(k), v_in=heads(v), cache=cache.struct()))
    ops.cache_read(gpu, ops.CacheReadArgs(dtype=hip.F32, rows=n, documents=1, kv_heads=1, head_dim=d, k_out=heads(out[0]),
                                          v_out=heads(out[1]), cache=cache.struct()))
    spread = x.unflatten(-1, (-1, 32))
    off = ((spread.amax(-1) - spread.amin(-1)).double() / 30 + 92).repeat_interleave(32, -1)
    for got, want in ((out[0], x), (out[1], -x)):
        assert bool(torch.isfinite(got).all())
        assert bool(((got[:, 0].double() - want.double()).abs() <= off).all())
