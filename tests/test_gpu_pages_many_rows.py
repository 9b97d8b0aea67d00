"""Pools of more sequences than the one workgroup of a reserve has threads (several rows a thread), up to the most that a pool takes, against
oracle/q4_oracle.py; whole numbers and bytes, so everything has to be equal."""
import numpy as np
import pytest
import torch

from oracle import q4_oracle as Q

gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("W,n,P,block", [(1025, 3, 2100, 8), (1500, 9, 4000, 4), (2731, 5, 7000, 16), (4095, 1, 4100, 8), (4096, 2, 5000, 8), (4096, 7, 20000, 2)])
def test_pools_of_many_rows(W, n, P, block):
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(W + n)
    table, lengths, refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
    data = rng.integers(0, 256, (P, 20), dtype=np.uint8)
    t, l, r, c = ints(table), ints(lengths), ints(refs), torch.tensor(data).cuda()

    def same(what):
        for a, b in ((t, table), (l, lengths), (r, refs), (c, data)):
            assert (a.cpu().numpy() == b).all(), what

    def reserve(n_new, what):
        got = A.reserve_blocks(t, l, r, ints(n_new), [c], block)
        want, copies = Q.reserve(table, lengths, refs, n_new, block)
        for s, d in copies:
            data[d] = data[s]
        assert (got.cpu().numpy() == want).all(), what
        same(what)

    for step in range(3):
        reserve(np.where(rng.random(W) < 0.3, rng.integers(0, block + 3, W), 0), (step, "some"))
        parents = np.where(rng.random(W) < 0.5, np.arange(W), rng.integers(-1, W + 1, W))
        A.fork_blocks(t, l, r, ints(parents), block)
        Q.fork(table, lengths, refs, parents, block)
        same((step, "fork"))
        lengths[:] = np.where(rng.random(W) < 0.2, lengths // block * block, np.where(rng.random(W) < 0.2, lengths // 2, lengths))
        l.copy_(ints(lengths))
        reserve(np.ones(W, int), (step, "one each"))
        finished = rng.random(W) < 0.4
        A.free_blocks(t, l, r, torch.tensor(finished).cuda())
        Q.fork(table, lengths, refs, np.where(finished, -1, np.arange(W)), block)
        same((step, "free"))
        used = A.compact_blocks(t, r, [c])
        want, moves = Q.compact(table, refs)
        for s, d in moves:
            data[d] = data[s]
        assert int(used) == want
        same((step, "compact"))


@gpu
def test_one_page_shared_by_all_rows():
    """4096 continuations of one page: each but the last asks for a copy, as many as there are pages get one."""
    from inference_lib_amd import attention as A
    W, block, P = 4096, 8, 3000
    table, lengths, refs = np.full((W, 2), -1, np.int32), np.full(W, 5, np.int32), np.zeros(P, np.int32)
    table[:, 0] = 77
    refs[77] = W
    data = np.random.default_rng(0).integers(0, 256, (P, 48), dtype=np.uint8)
    t, l, r, c = ints(table), ints(lengths), ints(refs), torch.tensor(data).cuda()
    got = A.reserve_blocks(t, l, r, ints(np.ones(W)), [c], block)
    want, copies = Q.reserve(table, lengths, refs, np.ones(W, int), block)
    for s, d in copies:
        data[d] = data[s]
    assert len(copies) == P - 1 and (got.cpu().numpy() == want).all()
    for a, b in ((t, table), (l, lengths), (r, refs), (c, data)):
        assert (a.cpu().numpy() == b).all()
