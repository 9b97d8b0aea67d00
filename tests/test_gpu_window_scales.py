"""Scales at the ends of what the window attention takes: what is not seen has no weight, however small the scale."""
import math

import pytest

from test_gpu_window import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,heads", [("f32", (5, 5, 64)), ("f32", (4, 1, 128)), ("f16", (7, 1, 128)), ("bf16", (8, 2, 64)), ("bf16", (6, 1, 256))], ids=str)
@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -120, 2.0 ** -126, 2.0 ** -149])
@pytest.mark.parametrize("splits,row_blocks", [(0, 0), (1, 1), (3, 1), (2, 2), (1, 8), (4, 8)])
def test_least_scales(dtype, heads, scale, splits, row_blocks):
    """All logits are next to 0: a row's result is the mean of the values that it sees."""
    if (dtype == "f32" and row_blocks > 1) or (row_blocks == 2 and heads[2] == 256):
        pytest.skip("other row groups there")
    for S in (1, 3):
        b = Batch(dtype, *heads, [list(range(n - S, n)) for n in (S, 40, 333)], 50, 7, 16, seed=S, spread=scale * math.sqrt(heads[2]))
        b.check(b.fixed(splits, row_blocks), "fixed")
        b.check(b.packed(splits, row_blocks, behind=2), "packed")
