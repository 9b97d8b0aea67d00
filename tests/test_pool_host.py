"""Refusals of the operators on a pool's pages that need no GPU: every one of these returns before any work is queued."""
import ctypes as C

import pytest

from inference_lib_amd import _lib


@pytest.mark.parametrize("at", [0, 4, -4, 12, -12])
def test_positions_are_not_the_lengths(at):
    """reserve writes where the new tokens go and lets the lengths grow: in one tensor the positions would be lost."""
    p = _lib.HwPool()
    p.W, p.max_blocks, p.num_blocks, p.block_size = 4, 3, 8, 16
    p.block_table, p.seq_lengths, p.ref_counts = 4096, 65536, 8192
    n = C.c_size_t(0)
    assert _lib.lib.hw_pool_workspace_bytes(C.byref(p), C.byref(n)) == 0
    p.workspace, p.workspace_bytes = 16384, n.value
    assert _lib.lib.hw_reserve_blocks(C.byref(p), 12288, 65536 + at, None) == -3
