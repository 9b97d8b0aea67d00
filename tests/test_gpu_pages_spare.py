"""Pages that rows name behind their sequences' tokens: lengths that were shortened (drafts that were rejected, a return to a common prefix),
rows that were filled ahead.  Against oracle/q4_oracle.py; whole numbers and bytes, so everything has to be equal."""
import numpy as np
import pytest
import torch

from oracle import q4_oracle as Q

gpu = pytest.mark.gpu


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled_rows(rng, W, n, block, spare):
    """Every row names n pages of its own, with tokens in the first few of them."""
    P = W * n + spare
    table = rng.permutation(P)[: W * n].reshape(W, n).astype(np.int32)
    refs = np.zeros(P, np.int32)
    refs[table.ravel()] = 1
    return table, rng.integers(0, 3 * block, W).astype(np.int32), refs


@gpu
@pytest.mark.parametrize("W,n,block", [(64, 128, 16), (100, 80, 64), (8, 1000, 8), (64, 400, 16), (3, 3, 1)])
def test_pages_without_tokens_are_not_passed_on(W, n, block):
    """A row in every four forks, so most waves are done with the columns long before the others (one workgroup, and several)."""
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(W + n)
    for step in range(6):
        table, lengths, refs = filled_rows(rng, W, n, block, 7)
        t, l, r = ints(table), ints(lengths), ints(refs)
        who = np.arange(W)
        if step % 2 == 0:
            parents = np.where(who % 4 == 3, (who * 5 + step) % W, who)
            A.fork_blocks(t, l, r, ints(parents), block)
        else:
            finished = who % 4 == step % 4
            A.free_blocks(t, l, r, torch.tensor(finished).cuda())
            parents = np.where(finished, -1, who)
        Q.fork(table, lengths, refs, parents, block)
        assert (t.cpu().numpy() == table).all() and (l.cpu().numpy() == lengths).all() and (r.cpu().numpy() == refs).all(), step


def on_device(table, lengths, refs, data):
    return ints(table), ints(lengths), ints(refs), torch.tensor(data).cuda()


def same(dev, host, what):
    for a, b in zip(dev, host):
        assert (a.cpu().numpy() == b).all(), what


@gpu
@pytest.mark.parametrize("length,n_new", [(16, 1), (20, 1), (20, 20), (0, 64), (0, 1), (32, 9), (16, 17)])
@pytest.mark.parametrize("both", [False, True])
def test_reserve_behind_a_fork_and_a_shorter_length(length, n_new, both):
    """One or both of two sequences that share three pages of 16 go back, to a border and into a page."""
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(length + n_new)
    table = np.full((3, 4), -1, np.int32)
    table[0, :3] = table[2, :3] = [5, 1, 7]
    lengths, refs = np.array([length if both else 40, 0, length], np.int32), np.zeros(20, np.int32)
    refs[[5, 1, 7]] = 2
    data = rng.integers(0, 256, (20, 48), dtype=np.uint8)
    t, l, r, c = on_device(table, lengths, refs, data)
    ask = [n_new if both else 1, 3, n_new]
    got = A.reserve_blocks(t, l, r, ints(ask), [c], 16)
    want, copies = Q.reserve(table, lengths, refs, ask, 16)
    for s, d in copies:
        data[d] = data[s]
    same((got, t, l, r, c), (want, table, lengths, refs, data), (length, n_new, both))
    for w in range(3):                           # what is about to be written belongs to one sequence
        if want[w] < 64:
            assert all(refs[table[w, p // 16]] == 1 for p in range(want[w], lengths[w]))


@gpu
@pytest.mark.parametrize("seed,W,n,P,block", [(0, 6, 7, 34, 8), (1, 5, 40, 150, 1), (2, 70, 24, 500, 4), (3, 24, 300, 2500, 4), (4, 200, 60, 1700, 16), (5, 12, 40, 140, 2)])
def test_a_pool_whose_lengths_are_shortened_goes_the_way_of_the_oracle_s(seed, W, n, P, block):
    from inference_lib_amd import attention as A
    rng = np.random.default_rng(200 + seed)
    table, lengths, refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
    data = rng.integers(0, 256, (P, 20), dtype=np.uint8)
    t, l, r, c = on_device(table, lengths, refs, data)
    for step in range(24):
        kind = rng.choice(["fork", "shorter", "reserve", "reserve", "compact"])
        if kind == "fork":
            parents = np.where(rng.random(W) < 0.4, np.arange(W), rng.integers(-1, W, W))
            A.fork_blocks(t, l, r, ints(parents), block)
            Q.fork(table, lengths, refs, parents, block)
        elif kind == "shorter":
            to = (rng.random(W) * (lengths + 1)).astype(np.int32)
            to = np.where(rng.random(W) < 0.5, to // block * block, to)
            lengths[:] = np.where(rng.random(W) < 0.6, to, lengths)
            l.copy_(ints(lengths))
        elif kind == "reserve":
            n_new = rng.choice([0, 1, 1, 2, block, 3 * block + 1, 17 * block, int(rng.integers(0, max(2, n * block // 2)))], W)
            got = A.reserve_blocks(t, l, r, ints(n_new), [c], block)
            want, copies = Q.reserve(table, lengths, refs, n_new, block)
            for s, d in copies:
                data[d] = data[s]
            assert (got.cpu().numpy() == want).all(), step
        else:
            used = A.compact_blocks(t, r, [c])
            want, moves = Q.compact(table, refs)
            for s, d in moves:
                data[d] = data[s]
            assert int(used) == want
        same((t, l, r, c), (table, lengths, refs, data), (step, kind))
        assert (np.bincount(table[table >= 0], minlength=P) == refs).all()


@gpu
def test_positions_in_the_place_of_the_lengths_are_refused():
    from inference_lib_amd import attention as A
    t, l, r = ints([[0, -1]]), ints([3]), ints([1, 0])
    with pytest.raises(RuntimeError):
        A.reserve_blocks(t, l, r, ints([1]), [], 8, positions=l)
    assert l.tolist() == [3] and A.reserve_blocks(t, l, r, ints([1]), [], 8).tolist() == [3] and l.tolist() == [4]
