"""The heads' gradients over so many rows that a workgroup's take several batches
of sines, the last of them partial, against their formulas in 64 bits."""

import pytest

from beatlm_amd import ops
from tests.opsdata import DTYPES
from tests.test_gpu_heads import Heads, gpu  # noqa: F401

pytestmark = pytest.mark.gpu

# With 256 compute units a workgroup has ceil(rows / 768) rows, rounded up to the
# rows it holds at once. 25001 rows: 33. Of 16-bit heads of 256 it holds 16, and
# sines of 16 (2048 pairs): 48 rows, three batches. Of f32 heads 8 and 8 (1024):
# 40 rows, five. 13003 rows: 17; 1 + 2 heads in 16 bits go two at a time, 24 rows in
# batches of 16 and 8; of 255, an element at a time, three batches of 8.
SHAPES = [
    # rows, q_heads, k_heads, d, sections, neighbours, layout
    (25001, 1, 1, 256, [128], False, "qkv"), (25001, 1, 1, 256, [64, 64], True, "heads"), (13003, 1, 2, 256, [128], False, "qkv"), (13003, 1, 2, 255, [127], False, "odd"),
    (40010, 2, 1, 128, [64], True, "qkv"),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("norm", ["rms", "centred"])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_of_several_batches_of_sines(gpu, dtype, norm, shape):  # noqa: F811
    rows, q_heads, k_heads, d, sections, neighbours, layout = shape
    t = Heads(dtype, rows, q_heads, k_heads, d, sections, norm, neighbours, layout)
    ops.head_norm_rotary(gpu, t.table, t.args())
    ops.head_norm_rotary_backward(gpu, t.table, t.args(), t.grads(gpu))
    t.check()
