"""Infinite values that a row sees, where the rows of a group all see the same: steps of single tokens, at the positions that stand in for tokens
of their tile that nobody sees -- the last one, the last one of the window's first tile, the last sink -- and beside them."""
import math

import pytest
import torch

from test_gpu_window import Batch

pytestmark = pytest.mark.gpu
WINDOW, SINKS, BLOCK = 100, 20, 16
LENGTHS = (1, 7, 32, 33, 100, 130, 160, 333, 1000)              # the token at length - 1: positions inside and at the end of tiles, with and without a window to the left


class Infinite:
    """A batch with a few infinite values, those of every kv head at the positions and channels that `place` gives for a length as far as they
    are seen, and the same batch without."""

    def __init__(self, dtype, heads, place, S=1):
        self.wild, self.plain = (Batch(dtype, *heads, [[n - 1] * S for n in LENGTHS], WINDOW, SINKS, BLOCK, seed=heads[0]) for _ in range(2))
        for w, n in enumerate(LENGTHS):
            for value, j, e in place(n):
                if 0 <= j < n and (n - 1 - j < WINDOW or j < SINKS):
                    self.wild.vc[self.wild.table[w, j // BLOCK].long(), :, j % BLOCK, e] = value
        self.want, self.finite = self.wild.want()[0], self.plain.want()[0]
        assert not torch.isfinite(self.want).all()

    def check(self, got, what):
        """Infinite and NaN where the definition is; everything else as without such values, within its bounds."""
        out, lse = got
        there = ~torch.isfinite(self.want)
        assert torch.equal(torch.isnan(out), torch.isnan(self.want)), what
        assert torch.equal(torch.isinf(out), torch.isinf(self.want)) and torch.equal(out[torch.isinf(out)].double(), self.want[torch.isinf(out)]), what
        self.plain.check((torch.where(there, self.finite.to(out.dtype), out), lse), what)


PLACES = {
    "last": lambda n: [(math.inf, n - 1, 3)],
    "end of the first tile": lambda n: [(-math.inf, max(n - WINDOW, 0) // 32 * 32 + 31, 3)],
    "last sink": lambda n: [(math.inf, SINKS - 1, 3)],
    "first": lambda n: [(math.inf, max(n - WINDOW, 0), 3)],
    "all": lambda n: [(math.inf, n - 1, 3), (-math.inf, max(n - WINDOW, 0) // 32 * 32 + 31, 4), (math.inf, SINKS - 1, 5), (math.nan, n - 1, 6)],
}


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (7, 1, 128)), ("f32", (5, 5, 64)), ("f32", (4, 1, 128)), ("bf16", (6, 1, 256)), ("f16", (40, 1, 128))], ids=str)
@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("splits,row_blocks", [(0, 0), (1, 1), (3, 1), (1, 2), (2, 2), (1, 8), (5, 8)])
def test_seen_by_all_rows(dtype, heads, place, splits, row_blocks):
    if (dtype == "f32" and row_blocks > 1) or (row_blocks == 2 and heads[2] == 256):
        pytest.skip("other row groups there")
    b = Infinite(dtype, heads, PLACES[place])
    b.check(b.wild.fixed(splits, row_blocks), "fixed")
    b.check(b.wild.packed(splits, row_blocks, before=1, behind=3), "packed")


@pytest.mark.parametrize("dtype,heads", [("bf16", (8, 2, 64)), ("f16", (16, 2, 128)), ("bf16", (6, 2, 256))], ids=str)
@pytest.mark.parametrize("row_blocks", [0, 8])
def test_many_rows_at_one_position(dtype, heads, row_blocks):
    """Forty query tokens at one position: a group of many rows that all see the same."""
    b = Infinite(dtype, heads, PLACES["all"], S=40)
    b.check(b.wild.fixed(0, row_blocks), "fixed")
    b.check(b.wild.packed(0, row_blocks), "packed")
