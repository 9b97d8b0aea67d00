"""Pins of oracle/q4_oracle.py's pool where lengths are shortened between the steps (drafts that were rejected, a return to a common
prefix): whatever sequences share and give up, each one reads what it wrote.  CPU only."""
import numpy as np
import pytest

from oracle import q4_oracle as O


def counts(table, P):
    return np.array([(table == p).sum() for p in range(P)])


@pytest.mark.parametrize("bs", [1, 4, 8])
@pytest.mark.parametrize("seed", range(6))
def test_sequences_read_what_they_wrote(seed, bs):
    rng = np.random.default_rng(seed)
    W, n, P = 6, 7, 34
    table, lengths, refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
    data = np.full((P, bs), -1)                 # who wrote a position: (a token's number)
    content = [[] for _ in range(W)]
    number = 0
    for step in range(120):
        kind = rng.integers(0, 5)
        if kind == 0:
            parents = np.where(rng.random(W) < 0.5, np.arange(W), rng.integers(-1, W, W))
            O.fork(table, lengths, refs, parents, bs)
            content = [list(content[p]) if p >= 0 else [] for p in parents]
        elif kind == 1:
            _, moves = O.compact(table, refs)
            for s, d in moves:
                data[d] = data[s]
        elif kind == 2:                         # shorter: anything, or back to a page's border
            for w in range(W):
                if rng.random() < 0.6:
                    to = int(rng.integers(0, lengths[w] + 1))
                    lengths[w] = to if rng.random() < 0.5 else to // bs * bs
                    content[w] = content[w][: lengths[w]]
        else:
            most = int(rng.integers(1, 2 * bs + 2))
            n_new = rng.integers(0, most + 1, W)
            before = lengths.copy()
            pos, copies = O.reserve(table, lengths, refs, n_new, bs)
            for s, d in copies:
                data[d] = data[s]
            for w in range(W):
                if pos[w] >= n * bs:
                    assert lengths[w] == before[w]
                    continue
                assert pos[w] == before[w] and lengths[w] == before[w] + n_new[w]
                for t in range(most):           # (a batch padded to `most` tokens: what lies behind a sequence's own goes to pages of its own or nowhere)
                    p = int(pos[w]) + t
                    blk = int(table[w, p // bs]) if p < n * bs else -1
                    if t < n_new[w]:
                        assert blk >= 0
                    if blk >= 0:
                        assert refs[blk] == 1                    # nothing shared is written
                        data[blk, p % bs] = number
                    if t < n_new[w]:
                        content[w].append(number)
                    number += 1
        assert (counts(table, P) == refs).all()
        for w in range(W):
            got = [int(data[table[w, p // bs], p % bs]) for p in range(lengths[w])]
            assert got == content[w], (step, w)


def test_a_length_set_back_behind_a_fork():
    """Two rows of three pages of 16; one goes back to a border, or into a page, or to where its next tokens cover several pages."""
    def pool(len1):
        return np.array([[0, 1, 2, -1], [0, 1, 2, -1]], np.int32), np.array([40, len1], np.int32), np.array([2, 2, 2] + [0] * 6, np.int32)

    t, l, r = pool(16)
    pos, copies = O.reserve(t, l, r, [0, 1], 16)
    assert pos.tolist() == [64, 16] and copies == [] and l.tolist() == [40, 17]
    assert t.tolist() == [[0, 1, 2, -1], [0, 3, -1, -1]] and r.tolist() == [2, 1, 1, 1, 0, 0, 0, 0, 0]
    t, l, r = pool(20)
    pos, copies = O.reserve(t, l, r, [0, 20], 16)
    assert pos.tolist() == [64, 20] and copies == [(1, 3)]
    assert t.tolist() == [[0, 1, 2, -1], [0, 3, 4, -1]] and r.tolist() == [2, 1, 1, 1, 1, 0, 0, 0, 0]
    t, l, r = pool(0)
    pos, copies = O.reserve(t, l, r, [1, 64], 16)
    assert pos.tolist() == [40, 0] and copies == [(2, 3)]       # (the first is still one of two that name page 2 when both ask)
    assert t.tolist() == [[0, 1, 3, -1], [4, 5, 6, 7]] and r.tolist() == [1, 1, 0, 1, 1, 1, 1, 1, 0]
    t, l, r = pool(16)                                           # no page left: the row stays as it is
    r[3:] = 1
    pos, copies = O.reserve(t, l, r, [0, 1], 16)
    assert pos.tolist() == [64, 64] and l.tolist() == [40, 16] and t.tolist() == [[0, 1, 2, -1]] * 2 and r[:3].tolist() == [2, 2, 2]
