"""Refusals, plans and wrappers of the window attention, packed batches and drafts that need no GPU, and the oracle of their tests against
other ways to the same numbers."""
import ctypes as C
import math
import random

import numpy as np
import pytest
import torch

from inference_lib_amd import _lib
from inference_lib_amd import attention as A
from inference_lib_amd.cache import PagedCache
from oracle import window_oracle as wo


def problem(**over):
    p = _lib.HwWindowProblem()
    p.dtype, p.W, p.Hq, p.Hkv, p.D, p.S = _lib.HW_BF16, 2, 8, 2, 128, 1
    p.block_size, p.max_blocks, p.num_blocks, p.window, p.sinks, p.scale = 16, 4, 8, 40, 4, 0.1
    for f in ("out", "q", "locations", "key_cache", "value_cache", "block_table"):
        setattr(p, f, 4096)
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,status", [
    ({}, 0), (dict(dtype=5), -2), (dict(dtype=_lib.HW_F32), 0), (dict(dtype=_lib.HW_F32, D=256), -4), (dict(D=96), -4), (dict(D=0), -3), (dict(window=0), -3), (dict(window=-5), -3),
    (dict(sinks=-1), -3), (dict(window=(1 << 31) - 1, sinks=(1 << 31) - 1), 0), (dict(Hq=7), -3), (dict(W=0), -3), (dict(S=0), -3), (dict(S=4096), -3), (dict(scale=0.0), -3),
    (dict(scale=float("nan")), -3), (dict(block_size=0), -3), (dict(block_size=4096), -3), (dict(max_blocks=1 << 17), -3), (dict(num_blocks=1 << 28), -3), (dict(q=None), -1),
    (dict(locations=None), -1), (dict(key_cache=None), -1), (dict(block_table=None), -1), (dict(value_cache=4104), -7), (dict(out=4100), -7), (dict(splits=-1), -3), (dict(row_blocks=-1), -3),
    (dict(W=1 << 20), -3), (dict(cu_seqlens_q=4096, total_q=-1), -3), (dict(cu_seqlens_q=4096, total_q=1 << 19), -3), (dict(cu_seqlens_q=4096, total_q=0, q=None), 0),
])
def test_attention_refuses(over, status):
    p = problem(**over)
    assert _lib.lib.hw_window_validate(C.byref(p)) == status
    if status:
        fn = _lib.lib.hw_window_varlen_paged_sdpa if p.cu_seqlens_q else _lib.lib.hw_window_paged_sdpa
        assert fn(C.byref(p), None) == status
        assert _lib.lib.hw_window_plan_debug(C.byref(p), 256, C.byref(_lib.HwPagedPlan())) == status


def test_the_two_entries_keep_to_their_queries_and_null_arguments():
    lib, n = _lib.lib, C.c_size_t(0)
    assert lib.hw_window_paged_sdpa(C.byref(problem(cu_seqlens_q=4096)), None) == -3
    assert lib.hw_window_varlen_paged_sdpa(C.byref(problem()), None) == -1
    assert lib.hw_window_validate(None) == -1 and lib.hw_window_paged_sdpa(None, None) == -1 and lib.hw_window_varlen_paged_sdpa(None, None) == -1
    assert lib.hw_window_plan_debug(None, 256, C.byref(_lib.HwPagedPlan())) == -1 and lib.hw_window_workspace_bytes(None, C.byref(n)) == -1
    assert lib.hw_window_plan_debug(C.byref(problem()), 256, None) == -1 and lib.hw_window_plan_debug(C.byref(problem()), 0, C.byref(_lib.HwPagedPlan())) == -3
    assert lib.hw_packed_slots(None, None) == -1 and lib.hw_copy_to_slots(None, None) == -1 and lib.hw_trim_blocks(None, 1, 0, None) == -1
    assert lib.hw_verify_drafts(None, None) == -1 and lib.hw_verify_workspace_bytes(None, C.byref(n)) == -1


@pytest.mark.parametrize("over", [dict(dtype=_lib.HW_F32, row_blocks=2), dict(D=256, row_blocks=2), dict(row_blocks=3), dict(dtype=_lib.HW_F32, row_blocks=8)])
def test_row_blocks_that_no_kernel_has(over):
    assert _lib.lib.hw_window_plan_debug(C.byref(problem(**over)), 256, C.byref(_lib.HwPagedPlan())) == -4


def test_plans_of_random_problems():
    rng = random.Random(3)
    for _ in range(4000):
        Hkv, gq, D = rng.choice([1, 2, 3, 8, 16, 300]), rng.choice([1, 2, 5, 8, 24]), rng.choice([64, 128, 256])
        dtype = rng.choice([_lib.HW_F16, _lib.HW_BF16, _lib.HW_F32]) if D < 256 else _lib.HW_F16
        block = rng.randint(1, 300)
        kw = dict(W=rng.randint(1, 300), Hq=Hkv * gq, Hkv=Hkv, D=D, block_size=block, max_blocks=rng.randint(1, (1 << 20) // block), window=rng.choice([1, 40, 1000, 5000, (1 << 31) - 1]),
                  sinks=rng.choice([0, 4, 500, (1 << 31) - 1]), dtype=dtype, num_cus=rng.choice([1, 64, 256]), splits=rng.choice([0, 0, 0, 1, 7, 4000]))
        kw.update(dict(S=rng.randint(1, 60)) if rng.random() < 0.5 else dict(total_q=rng.randint(0, 9000)))
        tokens = kw["total_q"] if "total_q" in kw else kw["W"] * kw["S"]
        if tokens * gq >= 1 << 20:
            continue
        pl = _lib.window_plan(**kw)
        wide = pl.row_blocks == 8
        assert pl.rows == tokens * gq and pl.row_blocks in (1, 2, 8) and 1 <= pl.splits <= _lib.HW_MAX_SPLITS and not (wide and dtype == _lib.HW_F32)
        most = 16 * pl.row_blocks if not wide else 128 if D == 256 else 256
        if "S" in kw:
            assert pl.row_groups >= kw["W"] * -(-kw["S"] * gq // most) and pl.row_groups % kw["W"] == 0
        else:
            assert pl.row_groups > pl.rows // most or pl.rows == 0      # one more than the rows of any split into sequences need
            assert pl.row_groups >= kw["W"]
        if wide:
            assert pl.workgroups == Hkv * pl.splits and (pl.splits == 1 or pl.workspace_bytes == Hkv * (2 * pl.splits * most * (D + 2) * 4 + 16 * (1 + min(pl.row_groups, pl.splits * 7 // 8))))
        else:
            assert pl.workgroups == Hkv * pl.row_groups * pl.splits
            assert pl.workspace_bytes >= (0 if pl.splits == 1 else Hkv * pl.splits * pl.rows * (D + 2) * 4)


def test_row_groups_go_round_where_there_are_rows_for_it():
    """1024 tokens of 5 query heads a kv head: 32 groups for the 32 workgroups of each of 8 kv heads."""
    assert _lib.window_plan(W=1, Hq=40, Hkv=8, D=128, block_size=16, max_blocks=400, window=2048, num_cus=256, S=1024).row_groups == 32
    assert _lib.window_plan(W=1, Hq=40, Hkv=8, D=128, block_size=16, max_blocks=400, window=2048, num_cus=256, S=100).row_groups == 2


def packed(**over):
    b = _lib.HwPackedBatch()
    b.W, b.max_blocks, b.num_blocks, b.block_size, b.total = 2, 3, 8, 16, 5
    b.block_table = b.positions = b.n_new = b.cu_seqlens = b.locations = b.slots = 4096
    for k, v in over.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("over,status", [(dict(W=0), -3), (dict(W=4097), -4), (dict(max_blocks=0), -3), (dict(num_blocks=0), -3), (dict(block_size=0), -3), (dict(total=-1), -3), (dict(total=1 << 28), -3),
                                         (dict(block_size=1 << 30), -3), (dict(num_blocks=1 << 28), -3), (dict(positions=None), -1), (dict(slots=None), -1), (dict(cu_seqlens=None), -1)])
def test_packed_batches_refuse(over, status):
    assert _lib.lib.hw_packed_slots(C.byref(packed(**over)), None) == status


def copies(**over):
    c = _lib.HwCopySlots()
    c.dtype, c.total, c.Hkv, c.E, c.Ev, c.block_size, c.num_blocks = _lib.HW_F16, 3, 2, 64, 64, 16, 4
    c.key_states = c.value_states = c.key_cache = c.value_cache = c.slots = 4096
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("over,status", [(dict(dtype=9), -2), (dict(total=-1), -3), (dict(total=0, slots=None), 0), (dict(Hkv=0), -3), (dict(E=0), -3), (dict(block_size=0), -3), (dict(num_blocks=1 << 28), -3),
                                         (dict(E=1 << 16), -3), (dict(slots=None), -1), (dict(value_cache=None), -1)])
def test_copies_refuse(over, status):
    assert _lib.lib.hw_copy_to_slots(C.byref(copies(**over)), None) == status


def drafts(**over):
    v = _lib.HwVerify()
    v.dtype, v.token_bytes, v.W, v.K, v.V = _lib.HW_F32, 8, 2, 3, 50000
    v.drafts = v.target = v.draft_probs = v.uniforms = v.tokens = v.accepted = v.workspace = 4096
    v.workspace_bytes = 1 << 20
    for k, x in over.items():
        setattr(v, k, x)
    return v


@pytest.mark.parametrize("over,status", [(dict(dtype=3), -2), (dict(token_bytes=2), -2), (dict(W=-1), -3), (dict(W=0), 0), (dict(K=-1), -3), (dict(V=0), -3), (dict(V=1 << 30), -3), (dict(drafts=None), -1),
                                         (dict(target=None), -1), (dict(uniforms=None), -1), (dict(tokens=None), -1), (dict(accepted=None), -1), (dict(seq_lengths=4096), -1), (dict(workspace=None), -6),
                                         (dict(workspace_bytes=8), -6), (dict(workspace=4100), -6)])
def test_verification_refuses(over, status):
    assert _lib.lib.hw_verify_drafts(C.byref(drafts(**over)), None) == status


def test_trims_refuse():
    p = _lib.HwPool()
    p.W, p.max_blocks, p.num_blocks, p.block_size = 2, 3, 8, 16
    p.block_table = p.seq_lengths = p.ref_counts = 4096
    assert _lib.lib.hw_trim_blocks(C.byref(p), 0, 0, None) == -3 and _lib.lib.hw_trim_blocks(C.byref(p), 5, -1, None) == -3
    p.seq_lengths = None
    assert _lib.lib.hw_trim_blocks(C.byref(p), 5, 0, None) == -1


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = [("hw_window_problem", _lib.HwWindowProblem, ("scale", "out", "workspace", "row_blocks")), ("hw_packed_batch", _lib.HwPackedBatch, ("block_table", "slots")),
             ("hw_copy_slots", _lib.HwCopySlots, ("key_states", "vs_h", "slots")), ("hw_verify", _lib.HwVerify, ("drafts", "dp_k", "accepted", "workspace_bytes"))]
    lines = "".join(f'printf("%zu {" ".join("%zu" for _ in f)}\\n", sizeof({c}), {", ".join(f"offsetof({c}, {x})" for x in f)});' for c, _, f in pairs)
    (tmp_path / "s.c").write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "hogwild_hip.h"\nint main(void) {{ {lines} return 0; }}\n')
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split("\n")
    for line, (_, t, f) in zip(out, pairs):
        assert [int(x) for x in line.split()] == [C.sizeof(t)] + [getattr(t, x).offset for x in f]


def test_python_wrappers_refuse_on_the_host():
    for kw in (dict(window=0), dict(window=-1), dict(window=8, sinks=-1), dict(sinks=4), dict(window=8, bits=4)):
        with pytest.raises(ValueError):
            PagedCache(1, 2, 64, 4, 2, device="cpu", **kw)
    with pytest.raises(ValueError):
        PagedCache(1, 2, 64, 4, 2, device="cpu").trim()
    with pytest.raises(ValueError):
        PagedCache(1, 2, 64, 4, 2, device="cpu", bits=4).reserve_packed(torch.ones(2, dtype=torch.int32), 2)
    cache = PagedCache(1, 2, 64, 4, 2, device="cpu", window=8, sinks=1)
    with pytest.raises(ValueError):
        cache.attend_packed(torch.zeros(3, 2, 64, dtype=torch.bfloat16), 0, 1.0)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)          # noqa: E731
    with pytest.raises(ValueError):
        A.packed_slots(ints(2, 3), ints(2), ints(2), 4, 16, 8, out=(ints(3), ints(5), ints(5)))
    for bad in (dict(n_new=ints(3)), dict(positions=ints(2).long()), dict(block_size=0), dict(slots=ints(5))):
        kw = dict(block_table=ints(2, 3), positions=ints(2), n_new=ints(2), cu_seqlens=ints(3), locations=ints(4), slots=ints(4), block_size=16, num_blocks=8)
        with pytest.raises(ValueError):
            _lib.packed_slots(**{**kw, **bad})
    k, c, s = torch.zeros(4, 2, 64), torch.zeros(8, 2, 16, 64), ints(4)
    for args in ((k[0], k[0], c, c, s), (k, k[:3], c, c, s), (k, k, c[:, :1], c[:, :1], s), (k, k, c.half(), c.half(), s), (k, k, c, c, s.long()), (k, k, c, c, ints(5)), (k, k, c.transpose(2, 3), c, s)):
        with pytest.raises(ValueError):
            _lib.copy_to_slots(*args)
    d, t, u = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4, 9), torch.zeros(2, 4)
    ok = dict(drafts=d, target_probs=t, uniforms=u)
    for bad in (dict(drafts=d[:, :2]), dict(drafts=d.float()), dict(target_probs=t[:, :3]), dict(uniforms=u.double()), dict(uniforms=u[:, :3]), dict(draft_probs=t), dict(draft_probs=t[:, :3].half()),
                dict(n_drafts=ints(3)), dict(positions=ints(2)), dict(seq_lengths=ints(2)), dict(positions=ints(2), seq_lengths=ints(2).long())):
        with pytest.raises(ValueError):
            _lib.verify_drafts(**{**ok, **bad})
    q, loc, table = torch.zeros(2, 4, 1, 64), ints(2, 1), ints(2, 3)
    ok = dict(q=q, locations=loc, key_cache=c, value_cache=c, block_table=table, scale=1.0, window=5, sinks=0, out=torch.zeros_like(q))
    for bad in (dict(window=0), dict(sinks=-1), dict(window=1 << 31), dict(locations=ints(2, 2)), dict(q=q.half()), dict(block_table=table.long()), dict(value_cache=c[:4]), dict(out=torch.zeros(3, 4, 1, 64), q=torch.zeros(3, 4, 1, 64)),
                dict(cu_seqlens_q=ints(3)), dict(lse=torch.zeros(2, 4)), dict(key_cache=c[..., :32], value_cache=c[..., :32])):
        with pytest.raises(ValueError):
            _lib.WindowProblem(**{**ok, **bad})


# ---- the oracle ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (7, 3), (16, 40), (100, 2)])
def test_oracle_attention_is_a_masked_softmax(window, sinks):
    g = torch.Generator().manual_seed(window)
    n, block, Hq, Hkv, D = 50, 8, 6, 2, 16
    row = torch.randperm(9, generator=g)[:7]
    kc, vc = torch.randn((9, Hkv, block, D), generator=g), torch.randn((9, Hkv, block, D), generator=g)
    q = torch.randn((n, Hq, D), generator=g)
    out, lse, *_ = wo.window_sdpa(q, list(range(n)), kc, vc, row, 0.3, window, sinks)
    k = kc[row].transpose(1, 2).reshape(-1, Hkv, D)[:n].double().repeat_interleave(Hq // Hkv, 1)
    v = vc[row].transpose(1, 2).reshape(-1, Hkv, D)[:n].double().repeat_interleave(Hq // Hkv, 1)
    a = 0.3 * torch.einsum("shd,nhd->shn", q.double(), k)
    i, j = torch.arange(n)[:, None], torch.arange(n)[None, :]
    a = a.masked_fill(~((j <= i) & ((i - j < window) | (j < sinks)))[:, None, :], -math.inf)
    assert torch.allclose(lse, torch.logsumexp(a, -1), atol=1e-12)
    assert torch.allclose(out, torch.einsum("shn,nhd->shd", torch.softmax(a, -1), v), atol=1e-12)
    nothing, none, *_ = wo.window_sdpa(q[:2], [-1, -7], kc, vc, row, 0.3, window, sinks)
    assert (nothing == 0).all() and (none == -math.inf).all()


def test_oracle_trims_what_no_later_token_sees():
    rng = np.random.default_rng(0)
    for window, sinks, block in [(1, 0, 4), (5, 3, 4), (9, 9, 3), (4, 100, 5)]:
        lengths = rng.integers(0, 60, 8).astype(np.int32)
        table = np.arange(8 * 20, dtype=np.int32).reshape(8, 20)
        refs = np.ones(8 * 20, dtype=np.int32)
        was = table.copy()
        wo.trim(table, lengths, refs, window, sinks, block)
        for w in range(8):
            later = {j for l in range(lengths[w], lengths[w] + 40) for j in wo.visible(l, window, sinks, 10 ** 6) if j < lengths[w]}
            for j in range(20):
                held = set(range(j * block, (j + 1) * block))
                gone = table[w, j] < 0
                assert gone == (held <= set(range(lengths[w])) and not held & later) and refs[was[w, j]] == (0 if gone else 1)


def test_oracle_verification_follows_the_target():
    """Three tokens, every draft and a fine grid of numbers: the token in the draft's place has the target's distribution."""
    p, q, n = torch.tensor([0.5, 0.125, 0.375]), torch.tensor([0.25, 0.5, 0.25]), 32
    u = (torch.arange(n) + 0.5) / n
    grid = torch.cartesian_prod(u, u)
    mass = torch.zeros(3, dtype=torch.float64)
    for x in range(3):
        W = grid.size(0)
        tokens, _ = wo.verify(torch.full((W, 1), x), p.expand(W, 2, 3), grid, q.expand(W, 1, 3))
        mass += q[x].double() * torch.bincount(tokens[:, 0], minlength=3).double() / W
    assert (mass - p.double()).abs().max() <= 1.0 / n
