"""Refusals and plans of the 4-bit caches and of the pages that need no GPU: every one of these returns before any work is queued."""
import ctypes as C

import pytest
import torch

from inference_lib_amd import _lib
from inference_lib_amd import attention as A


def copy_args(**over):
    c = _lib.HwCopyBlocks()
    c.dtype, c.B, c.Hkv, c.S_new, c.E, c.Ev = _lib.HW_F16, 1, 2, 1, 128, 128
    c.block_size, c.max_blocks, c.num_blocks = 16, 2, 4
    c.key_states = c.value_states = c.key_cache = c.value_cache = c.block_table = c.seq_lengths = 4096
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("fn", ["hw_copy_to_blocks_q4", "hw_read_blocks_q4"])
@pytest.mark.parametrize("over,status", [
    (dict(dtype=7), -2), (dict(E=64), -4), (dict(E=96, Ev=96), -4), (dict(E=512, Ev=512), -4), (dict(block_size=12), -3), (dict(block_size=0), -3),
    (dict(max_blocks=0), -3), (dict(num_blocks=0), -3), (dict(Hkv=0), -3), (dict(B=-1), -3), (dict(B=70000), -3), (dict(S_new=-1), -3),
    (dict(block_size=4096, max_blocks=1 << 20), -3), (dict(num_blocks=1 << 30), -3), (dict(key_cache=None), -1), (dict(seq_lengths=None), -1),
    (dict(key_cache=4100), -7), (dict(value_cache=4104), -7), (dict(B=0), 0), (dict(S_new=0), 0),
])
def test_append_and_read_refuse(fn, over, status):
    assert getattr(_lib.lib, fn)(C.byref(copy_args(**over)), None) == status


def test_null_arguments():
    lib = _lib.lib
    n = C.c_size_t(0)
    assert lib.hw_copy_to_blocks_q4(None, None) == -1 and lib.hw_read_blocks_q4(None, None) == -1
    assert lib.hw_paged_q4_validate(None) == -1 and lib.hw_paged_sdpa_q4(None, None) == -1 and lib.hw_varlen_paged_sdpa_q4(None, None) == -1
    assert lib.hw_paged_q4_plan_debug(None, 256, C.byref(_lib.HwPagedPlan())) == -1 and lib.hw_paged_q4_workspace_bytes(None, C.byref(n)) == -1
    assert lib.hw_pool_workspace_bytes(None, C.byref(n)) == -1 and lib.hw_fork_blocks(None, None, None) == -1 and lib.hw_free_blocks(None, None, None) == -1
    assert lib.hw_reserve_blocks(None, None, None, None) == -1 and lib.hw_compact_blocks(None, None, None) == -1


def paged(**over):
    p = _lib.HwPagedProblem()
    p.dtype, p.F, p.W, p.Hq, p.Hkv, p.E, p.Ev, p.S = _lib.HW_BF16, 1, 2, 8, 2, 128, 128, 1
    p.block_size, p.max_blocks, p.num_blocks, p.scale = 16, 4, 8, 0.1
    for f in ("out", "q", "locations", "fragment_lengths", "key_cache", "value_cache", "block_table"):
        setattr(p, f, 4096)
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,status", [
    ({}, 0), (dict(dtype=_lib.HW_F32), -4), (dict(dtype=5), -2), (dict(block_size=12), -3), (dict(block_size=4096), -3), (dict(E=64), -4), (dict(E=80, Ev=80), -4),
    (dict(F=0), -5), (dict(Hq=7), -3), (dict(scale=0.0), -3), (dict(scale=float("inf")), -3), (dict(S=0), -3), (dict(q=None), -1), (dict(key_cache=None), -1),
    (dict(key_cache=4104), -7), (dict(max_blocks=1 << 20), -3), (dict(num_blocks=1 << 28), -3),
])
def test_attention_refuses(over, status):
    assert _lib.lib.hw_paged_q4_validate(C.byref(paged(**over))) == status
    if status:
        assert _lib.lib.hw_paged_sdpa_q4(C.byref(paged(**over)), None) == status


def test_the_two_entries_keep_to_their_queries():
    assert _lib.lib.hw_paged_sdpa_q4(C.byref(paged(cu_seqlens_q=4096)), None) == -3
    assert _lib.lib.hw_varlen_paged_sdpa_q4(C.byref(paged()), None) == -1


@pytest.mark.parametrize("kw", [dict(W=1, S=1, Hq=8, Hkv=2, Ev=64, block_size=8, max_blocks=1), dict(W=4, S=1, Hq=40, Hkv=8, Ev=128, block_size=16, max_blocks=783),
                                dict(W=1, S=4000, Hq=64, Hkv=8, Ev=128, block_size=64, max_blocks=100), dict(W=64, S=1, Hq=16, Hkv=8, Ev=256, block_size=32, max_blocks=500),
                                dict(W=3, total_q=0, Hq=8, Hkv=8, Ev=64, block_size=8, max_blocks=9), dict(W=300, total_q=5000, Hq=32, Hkv=8, Ev=128, block_size=16, max_blocks=300)])
def test_plans_cover_the_rows(kw):
    pl = _lib.paged_plan(num_cus=256, q4=True, **kw)
    tokens = kw["total_q"] if "total_q" in kw else kw["W"] * kw["S"]
    assert pl.rows == tokens * kw["Hq"] // kw["Hkv"] and pl.splits >= 1 and pl.row_blocks >= 1
    assert pl.workgroups >= kw["Hkv"] and pl.workspace_bytes > 0
    if "S" in kw:
        assert pl.row_groups * 16 * pl.row_blocks * kw["W"] >= pl.rows


def test_plans_of_random_problems():
    import random
    rng = random.Random(5)
    for _ in range(3000):
        Hkv = rng.choice([1, 2, 3, 8, 16])
        kw = dict(W=rng.randint(1, 300), Hq=Hkv * rng.choice([1, 2, 5, 8]), Hkv=Hkv, Ev=rng.choice([64, 128, 256]), block_size=8 * rng.randint(1, 64))
        kw["max_blocks"] = rng.randint(1, max(1, min(3000, (1 << 20) // kw["block_size"])))
        if rng.random() < 0.5:
            kw["S"] = rng.randint(1, 40)
        else:
            kw["total_q"] = rng.randint(1, 9000)
        try:
            pl = _lib.paged_plan(num_cus=256, q4=True, **kw)
        except _lib.HogwildError:
            assert (kw.get("total_q") or kw["W"] * kw["S"]) * kw["Hq"] // Hkv >= 1 << 14      # more workgroups than a launch takes
            continue
        rows = (kw.get("total_q") or kw["W"] * kw["S"]) * kw["Hq"] // Hkv
        tiles = (kw["block_size"] * kw["max_blocks"] + 31) // 32
        assert pl.rows == rows and pl.row_blocks in (1, 2) and (kw["Ev"] < 256 or pl.row_blocks == 1)
        assert pl.workgroups == Hkv * pl.row_groups * pl.splits < 1 << 20
        assert 1 <= pl.splits <= max(1, min(64, (tiles + 3) // 4)) and (tiles > 24 or pl.splits == 1 or tiles > 12)
        assert pl.workspace_bytes >= Hkv * pl.splits * rows * (kw["Ev"] + 2) * 4
        groups = kw["W"] * -(-kw["S"] * kw["Hq"] // Hkv // (16 * pl.row_blocks)) if "S" in kw else kw["W"] + rows // (16 * pl.row_blocks)
        assert pl.row_groups >= min(groups, rows)


def pool(**over):
    p = _lib.HwPool()
    p.W, p.max_blocks, p.num_blocks, p.block_size = 2, 3, 8, 16
    p.block_table = p.seq_lengths = p.ref_counts = 4096
    ptr, size = (C.c_void_p * 1)(4096), (C.c_size_t * 1)(64)
    p.caches, p.page_bytes, p.n_caches = C.cast(ptr, C.POINTER(C.c_void_p)), C.cast(size, C.POINTER(C.c_size_t)), 1
    for k, v in over.items():
        setattr(p, k, v)
    return p, (ptr, size)


@pytest.mark.parametrize("over,status", [
    (dict(W=0), -3), (dict(W=4097), -4), (dict(max_blocks=0), -3), (dict(num_blocks=0), -3), (dict(block_size=0), -3), (dict(block_size=1 << 30), -3),
    (dict(num_blocks=1 << 29), -3), (dict(block_table=None), -1), (dict(ref_counts=None), -1), (dict(n_caches=-1), -3), ({}, -6), (dict(workspace=4096, workspace_bytes=8), -6),
])
def test_pools_refuse(over, status):
    p, keep = pool(**over)
    assert _lib.lib.hw_reserve_blocks(C.byref(p), 4096, 4096, None) == status
    assert _lib.lib.hw_compact_blocks(C.byref(p), 4096, None) == status
    assert _lib.lib.hw_fork_blocks(C.byref(p), None, None) < 0 and _lib.lib.hw_free_blocks(C.byref(p), None, None) < 0
    assert _lib.lib.hw_reserve_blocks(C.byref(p), None, 4096, None) < 0 and _lib.lib.hw_compact_blocks(C.byref(p), None, None) < 0


def test_copies_refuse_pages_named_twice_and_outside():
    ptr, size = (C.c_void_p * 2)(4096, 8192), (C.c_size_t * 2)(64, 0)
    run = lambda n_caches, s, d, n=None: _lib.lib.hw_copy_pages(ptr, size, n_caches, 8, (C.c_int32 * 8)(*s), (C.c_int32 * 8)(*d), len(s) if n is None else n, None)   # noqa: E731
    assert run(1, [0, 1], [2, 2]) == -3 and run(1, [0, 2], [2, 3]) == -3 and run(1, [0], [0]) == -3 and run(1, [8], [1]) == -3 and run(1, [1], [-1]) == -3
    assert run(2, [0], [1]) == -3 and run(1, [0], [1], n=-1) == -3 and run(1, [0], [1], n=9) == -3 and run(1, [], []) == 0 and run(0, [0], [1]) == 0


def test_python_wrappers_refuse_on_the_host():
    with pytest.raises(ValueError):
        A.q4_cache(4, 2, 12, 128, device="cpu")
    with pytest.raises(ValueError):
        A.copy_blocks([], [0], [1])
    c = torch.zeros(4, 8)
    for s, d in (([0], [4]), ([0, 1], [2]), ([-1], [2])):
        with pytest.raises(ValueError):
            A.copy_blocks([c], s, d)
    from inference_lib_amd.cache import PagedCache
    for kw in (dict(bits=8), dict(bits=16, dtype=torch.float32), dict(bits=4, block_size=12)):
        with pytest.raises(ValueError):
            PagedCache(1, 2, 128, 4, 2, device="cpu", **kw)
    assert PagedCache(2, 2, 64, 4, 3, device="cpu", bits=4).keys[0].shape == (4, 2, 16, 36)
