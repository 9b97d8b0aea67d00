"""Refusals of packed steps and their verification that need no GPU."""
import ctypes as C

import pytest
import torch

from inference_lib_amd import _lib


def ints(*s):
    return torch.zeros(s, dtype=torch.int32)


def pool():
    p, n = _lib.HwPool(), C.c_size_t(0)
    p.W, p.max_blocks, p.num_blocks, p.block_size = 4, 3, 8, 16
    p.block_table, p.seq_lengths, p.ref_counts = 65536, 8192, 32768
    assert _lib.lib.hw_pool_workspace_bytes(C.byref(p), C.byref(n)) == 0
    p.workspace, p.workspace_bytes = 1 << 20, n.value
    return p


@pytest.mark.parametrize("bad", [dict(n_new=ints(2)), dict(n_new=ints(2), positions=ints(2)), dict(n_new=ints(3), positions=ints(2), seq_lengths=ints(2)),
                                 dict(n_new=ints(2).long(), positions=ints(2), seq_lengths=ints(2)), dict(n_new=ints(4)[::2], positions=ints(2), seq_lengths=ints(2))])
def test_numbers_of_new_tokens_go_with_the_lengths(bad):
    with pytest.raises(ValueError):
        _lib.verify_drafts(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4, 9), torch.zeros(2, 4), **bad)


@pytest.mark.parametrize("taken,total,status", [(None, 5, -1), (49152, 1 << 28, -3), (49152, (1 << 31) - 1, -3)])
def test_rows_of_a_batch(taken, total, status):
    p = pool()
    assert _lib.lib.hw_reserve_step(C.byref(p), 4096, total, 16384, taken, None) == status


@pytest.mark.parametrize("total,positions", [(-2, ints(2, 2)), (1 << 28, ints(2, 2)), (4, ints(2))])
def test_reserve_refuses_other_totals(total, positions):
    with pytest.raises(ValueError):
        _lib.reserve_blocks(ints(2, 5), ints(2), ints(9), ints(2), positions, [], 16, total)


@pytest.mark.parametrize("taken,status", [(None, -1), (4096, -3), (4112 - 4, -3), (8192 + 12, -3), (16384 - 12, -3)])
def test_numbers_taken_lie_apart(taken, status):
    """Not in the new tokens' numbers, the positions or the lengths, nor across them."""
    p = pool()
    assert _lib.lib.hw_reserve_step(C.byref(p), 4096, -1, 16384, taken, None) == status


@pytest.mark.parametrize("positions", [ints(3), ints(3, 2), ints(1, 2), ints(2, 3), ints(2, 2).long(), ints(2, 4)[:, ::2]])
def test_reserve_refuses_other_positions(positions):
    with pytest.raises(ValueError):
        _lib.reserve_blocks(ints(2, 5), ints(2), ints(9), ints(2), positions, [], 16)


def test_more_workgroups_than_a_launch_takes():
    """Refused with a status of their own, before anything reaches the device."""
    c = _lib.HwCopySlots()
    c.dtype, c.Hkv, c.E, c.Ev, c.block_size, c.num_blocks = _lib.HW_F16, 1, 1, 1, 16, 4
    c.key_states = c.value_states = c.key_cache = c.value_cache = c.slots = 4096
    for total in (1 << 25, 1 << 26, (1 << 31) - 1):
        c.total = total
        assert _lib.lib.hw_copy_to_slots(C.byref(c), None) == -3
    v, n = _lib.HwVerify(), C.c_size_t(0)
    v.dtype, v.token_bytes, v.K = _lib.HW_F32, 8, 1
    for W, V in [(1 << 22, 2), (1 << 20, 1 << 16), (1 << 12, 1 << 24), ((1 << 31) - 1, 4096)]:
        v.W, v.V = W, V
        assert _lib.lib.hw_verify_workspace_bytes(C.byref(v), C.byref(n)) == -3 and _lib.lib.hw_verify_drafts(C.byref(v), None) == -3
    v.W, v.V = (1 << 22) - 1, 4096
    assert _lib.lib.hw_verify_workspace_bytes(C.byref(v), C.byref(n)) == 0 and n.value == 0
    v.W, v.V = (1 << 20) - 1, 1 << 16
    assert _lib.lib.hw_verify_workspace_bytes(C.byref(v), C.byref(n)) == 0 and n.value > 0
