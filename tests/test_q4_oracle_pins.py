"""Pins of oracle/q4_oracle.py: the quantiser and the layout against literal loops, the pages against what a pool has to keep."""
import math

import numpy as np
import pytest

from oracle import q4_oracle as O


def test_quantiser_element_by_element():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((3, 128)) * [[1.0], [100.0], [1e-3]]).astype(np.float32)
    code, scale, offset = O.quantise(x)
    for i in range(3):
        for g in range(2):
            part = x[i, 64 * g: 64 * g + 64]
            m = np.float32(np.float16(min(part)))
            s = np.float32(np.float16(np.float32(np.float32(max(part)) - m) / np.float32(15)))
            assert np.float32(offset[i, g]) == m and np.float32(scale[i, g]) == s
            for e in range(64):
                q = (float(part[e]) - float(m)) / float(s)
                want = min(15, max(0, math.floor(q + 0.5) if abs(q - round(q)) != 0.5 else 2 * round(q / 2)))
                assert code[i, 64 * g + e] == want
    # half a step, the step's own rounding (15 steps of it) and the offset's
    v = O.values(code, scale, offset)
    s, m = np.repeat(scale.astype(np.float64), 64, -1), np.repeat(offset.astype(np.float64), 64, -1)
    assert (np.abs(v - x) <= s * (0.5 + 15 * 2.0 ** -11) + np.abs(m) * 2.0 ** -11 + 1e-7).all()


def test_values_that_are_not_finite_or_too_large():
    x = np.zeros((4, 64), np.float32)
    x[0, 3], x[0, 4] = np.nan, 2.0
    x[1, 0], x[1, 1] = np.inf, -np.inf
    x[2, 0] = 1e30
    x[3] = 0.1
    v = O.values(*O.quantise(x))
    assert np.isfinite(v.astype(np.float16)).all()
    assert v[0, 3] == 0 and abs(v[0, 4] - 2) < 2e-3
    assert v[1, 1] == -65024 and abs(v[1, 0] - 65024) < 100 and abs(v[2, 0] - 65024) < 100
    # whatever the rounding of scale and offset, a value fits fp16
    rng = np.random.default_rng(3)
    big = (rng.uniform(-1, 1, (4000, 64)) * 10 ** rng.uniform(3, 6, (4000, 1)) + 10 ** rng.uniform(3, 6, (4000, 1))).astype(np.float32)
    assert np.isfinite(O.values(*O.quantise(big)).astype(np.float16)).all()
    assert (v[3] == v[3, 0]).all() and abs(v[3, 0] - 0.1) <= 0.1 * 2.0 ** -11      # a group of one value: the offset, and what its scale can add


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("keys", [True, False])
def test_layout_is_one_to_one_and_what_the_header_says(D, keys):
    byte, shift = O.code_place(D, keys)
    assert len({(b, s) for b, s in zip(byte.ravel(), shift.ravel())}) == 8 * D and byte.max() == 4 * D - 1
    s_at, m_at = O.param_place(D)
    assert sorted(np.concatenate([s_at.ravel(), s_at.ravel() + 1, m_at.ravel(), m_at.ravel() + 1])) == list(range(4 * D, 8 * O.row_bytes(D)))
    for t in range(8):                          # the sentence of the header, word by word
        for w in range(D // 8 if keys else D):
            for i in range(8):
                e = 2 * i if i < 4 else 2 * i - 7
                if keys:
                    r = w % (D // 32)
                    c, tok, word = 64 * (r // 2) + 16 * (w // (D // 32)) + 8 * (r % 2) + e, t, t * (D // 8) + w
                else:
                    c, tok, word = w, e, w
                assert byte[tok, c] == word * 4 + i // 2 and shift[tok, c] == 4 * (i % 2)


def test_a_token_is_read_as_it_was_written_and_the_others_stay():
    rng = np.random.default_rng(1)
    for D in (64, 128):
        for keys in (True, False):
            o = rng.integers(0, 256, 8 * O.row_bytes(D), dtype=np.uint8)
            o[4 * D:] = np.frombuffer(np.ones(len(o[4 * D:]) // 2, np.float16).tobytes(), np.uint8)
            before = O.read_octet(o, D, keys)
            x = rng.standard_normal(D).astype(np.float32)
            O.write_token(o, 5, x, keys)
            after = O.read_octet(o, D, keys)
            assert (after[5] == O.values(*O.quantise(x))).all()
            assert (np.delete(after, 5, 0) == np.delete(before, 5, 0)).all()


def counts(table, P):
    return np.array([(table == p).sum() for p in range(P)])


@pytest.mark.parametrize("seed", range(8))
def test_pages_keep_their_invariants(seed):
    rng = np.random.default_rng(seed)
    W, n, P, bs = 6, 7, 30, 8
    table, lengths, refs = np.full((W, n), -1, np.int32), np.zeros(W, np.int32), np.zeros(P, np.int32)
    data = np.full((P, bs), -1)                 # who wrote a position: (a token's number)
    content = [[] for _ in range(W)]
    number = 0
    for step in range(60):
        kind = rng.integers(0, 4)
        if kind == 0:
            parents = np.where(rng.random(W) < 0.5, np.arange(W), rng.integers(-1, W, W))
            O.fork(table, lengths, refs, parents, bs)
            content = [list(content[p]) if p >= 0 else [] for p in parents]
        elif kind == 1:
            n_used, moves = O.compact(table, refs)
            for s, d in moves:
                data[d] = data[s]
            assert (refs[:n_used] > 0).all() and (refs[n_used:] == 0).all()
        else:
            n_new = rng.integers(0, 12, W)
            before = lengths.copy()
            pos, copies = O.reserve(table, lengths, refs, n_new, bs)
            for s, d in copies:
                data[d] = data[s]
            for w in range(W):
                if pos[w] < n * bs:
                    assert pos[w] == before[w] and lengths[w] == before[w] + n_new[w]
                    for t in range(n_new[w]):
                        p = int(pos[w]) + t
                        blk = table[w, p // bs]
                        assert refs[blk] == 1                        # nothing shared is written
                        data[blk, p % bs] = number
                        content[w].append(number)
                        number += 1
                else:
                    assert lengths[w] == before[w]
        assert (counts(table, P) == refs).all()
        for w in range(W):                      # every sequence reads what it wrote, whatever the others did
            got = [int(data[table[w, p // bs], p % bs]) for p in range(lengths[w])]
            assert got == content[w]
